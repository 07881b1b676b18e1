// Python bindings of the mixture-of-experts kernels and of the 8-bit activation checkpoints.  Outputs are allocated here; in the
// poison mode (ops/debug.py) `track` gets each before its kernel runs.  Every call returns the number of kernels it launched last.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "bind_common.h"
#include "moe_api.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

struct Outputs {
  const pybind11::object& track;
  Tensor operator()(const char* name, c10::IntArrayRef size, const at::TensorOptions& options) const {
    Tensor t = torch::empty(size, options);
    if (!track.is_none()) track(name, t);
    return t;
  }
};

const __nv_bfloat16* bf(const Tensor& t) { return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()); }
__nv_bfloat16* bfm(const Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

bool bf16_or_f32(const Tensor& t, const char* what) {
  const bool b = t.scalar_type() == torch::kBFloat16;
  TORCH_CHECK(b || t.scalar_type() == torch::kFloat32, what, ": bf16 or fp32 expected, got ", t.scalar_type());
  return b;
}
// A matrix on the GPU whose rows are contiguous
void check_rows(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), what, ": a 2-D CUDA tensor with contiguous rows expected");
  TORCH_CHECK(t.size(0) < (1ll << 31) && t.size(1) < (1ll << 31), what, ": sizes of 2^31 and more are not supported");
}
void check_bf16(const Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, what, ": bf16 expected, got ", t.scalar_type());
}
void check_ints(const Tensor& t, int64_t n, const Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kInt32 && t.is_contiguous() && t.numel() == n, what, ": contiguous int32 of ", n,
              " elements on the GPU expected");
  TORCH_CHECK(t.device() == like.device(), what, ": on another GPU than its operand");
}
int64_t blocks_of(int64_t n) { return (n + tb::kActBlock - 1) / tb::kActBlock; }

struct Routed {
  Tensor weights, experts, slots, offsets, rows, counts, aux;
};

Routed do_route(const Tensor& logits, int64_t k, int64_t capacity, const Outputs& make) {
  check_rows(logits, "route");
  const bool b16 = bf16_or_f32(logits, "route: logits");
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= tb::kMaxExperts, "route: 1 to ", tb::kMaxExperts, " experts, got ", E);
  TORCH_CHECK(k >= 1 && k <= E && k <= tb::kMaxChoices, "route: top_k of ", k, " among ", E, " experts (at most ", tb::kMaxChoices, ")");
  TORCH_CHECK(capacity >= 0 && capacity < (1ll << 31), "route: capacity ", capacity);
  TORCH_CHECK(T * k <= (1ll << 30), "route: too many choices");
  const auto f32 = logits.options().dtype(torch::kFloat32), i32 = logits.options().dtype(torch::kInt32);
  Routed r;
  r.weights = make("route.weights", {T, k}, f32);
  r.aux = make("route.aux", {}, f32);
  r.experts = torch::empty({T, k}, i32);
  r.slots = torch::empty({T, k}, i32);
  r.rows = torch::empty({T * k}, i32);
  if (T == 0) {
    r.offsets = torch::zeros({E + 1}, i32);
    r.counts = torch::zeros({E}, i32);
    r.aux.zero_();
    return r;
  }
  // offsets, counts and scratch of one allocation
  const int64_t scratch = tb::route_scratch_ints((int)T, (int)E);
  Tensor ints = torch::empty({2 * E + 1 + scratch}, i32);
  r.offsets = ints.narrow(0, 0, E + 1);
  r.counts = ints.narrow(0, E + 1, E);
  const int rc = tb::route_fwd(logits.data_ptr(), b16, logits.stride(0), (int)T, (int)E, (int)k, (int)capacity, r.weights.data_ptr<float>(),
                               r.experts.data_ptr<int>(), r.slots.data_ptr<int>(), r.offsets.data_ptr<int>(), r.rows.data_ptr<int>(),
                               r.counts.data_ptr<int>(), r.aux.data_ptr<float>(), ints.data_ptr<int>() + 2 * E + 1, cur_stream());
  TORCH_CHECK(rc == 0, "route failed with code ", rc);
  return r;
}

Tensor do_route_bwd(const Tensor& logits, const Tensor& weights, const Tensor& experts, const Tensor& counts, const OptTensor& dweights,
                    const OptTensor& daux, const Outputs& make) {
  check_rows(logits, "route_bwd");
  const bool b16 = bf16_or_f32(logits, "route_bwd: logits");
  const int64_t T = logits.size(0), E = logits.size(1), k = weights.size(1);
  check_ints(experts, T * k, logits, "route_bwd: experts");
  check_ints(counts, E, logits, "route_bwd: counts");
  TORCH_CHECK(weights.scalar_type() == torch::kFloat32 && weights.is_contiguous() && weights.numel() == T * k, "route_bwd: weights");
  TORCH_CHECK(!has(dweights) || (dweights->scalar_type() == torch::kFloat32 && dweights->is_contiguous() && dweights->numel() == T * k),
              "route_bwd: dweights");
  TORCH_CHECK(!has(daux) || (daux->is_cuda() && daux->scalar_type() == torch::kFloat32 && daux->numel() == 1), "route_bwd: daux");
  Tensor dl = make("route_bwd", {T, E}, logits.options());
  if (T == 0) return dl;
  const int rc = tb::route_bwd(logits.data_ptr(), b16, logits.stride(0), weights.data_ptr<float>(), experts.data_ptr<int>(),
                               counts.data_ptr<int>(), has(dweights) ? dweights->data_ptr<float>() : nullptr,
                               has(daux) ? daux->data_ptr<float>() : nullptr, dl.data_ptr(), (int)T, (int)E, (int)k, cur_stream());
  TORCH_CHECK(rc == 0, "route_bwd failed with code ", rc);
  return dl;
}

Tensor do_gather(const Tensor& x, const Tensor& rows, int64_t k, const Outputs& make) {
  check_rows(x, "dispatch");
  const bool b16 = bf16_or_f32(x, "dispatch");
  const int64_t T = x.size(0), D = x.size(1), R = rows.numel();
  check_ints(rows, R, x, "dispatch: rows");
  Tensor out = make("dispatch", {R, D}, x.options().dtype(torch::kBFloat16));
  tb::rows_gather(x.data_ptr(), b16, x.stride(0), rows.data_ptr<int>(), bfm(out), (int)T, (int)k, (int)R, (int)D, cur_stream());
  return out;
}

Tensor do_combine(const Tensor& y, const OptTensor& weights, const Tensor& slots, at::ScalarType type, const Outputs& make) {
  check_rows(y, "combine");
  check_bf16(y, "combine");
  TORCH_CHECK(y.is_contiguous(), "combine: contiguous rows expected");
  const int64_t T = slots.size(0), k = slots.size(1), R = y.size(0), D = y.size(1);
  check_ints(slots, T * k, y, "combine: slots");
  TORCH_CHECK(!has(weights) || (weights->scalar_type() == torch::kFloat32 && weights->is_contiguous() && weights->numel() == T * k &&
                                weights->device() == y.device()), "combine: weights must be contiguous fp32 [tokens, choices]");
  TORCH_CHECK(type == torch::kBFloat16 || type == torch::kFloat32, "combine: bf16 or fp32 output");
  Tensor out = make("combine", {T, D}, y.options().dtype(type));
  tb::rows_combine(bf(y), has(weights) ? weights->data_ptr<float>() : nullptr, slots.data_ptr<int>(), out.data_ptr(),
                   type == torch::kBFloat16, (int)T, (int)k, (int)R, (int)D, cur_stream());
  return out;
}

std::tuple<Tensor, Tensor> combine_bwd(const Tensor& dout, const Tensor& y, const Tensor& weights, const Tensor& slots,
                                       const Tensor& offsets, const pybind11::object& track) {
  const Outputs make{track};
  check_rows(dout, "combine_bwd");
  const bool b16 = bf16_or_f32(dout, "combine_bwd");
  const int64_t T = slots.size(0), k = slots.size(1), D = y.size(1), E = offsets.numel() - 1;
  check_rows(y, "combine_bwd: y");
  check_bf16(y, "combine_bwd: y");
  TORCH_CHECK(y.is_contiguous() && y.size(0) == T * k && dout.size(0) == T && dout.size(1) == D, "combine_bwd: shapes");
  check_ints(slots, T * k, y, "combine_bwd: slots");
  check_ints(offsets, E + 1, y, "combine_bwd: offsets");
  TORCH_CHECK(weights.scalar_type() == torch::kFloat32 && weights.is_contiguous() && weights.numel() == T * k, "combine_bwd: weights");
  c10::cuda::CUDAGuard guard(y.device());
  Tensor dy = make("combine_bwd.dy", {T * k, D}, y.options());
  Tensor dw = make("combine_bwd.dweights", {T, k}, weights.options());
  tb::rows_combine_bwd(dout.data_ptr(), b16, dout.stride(0), bf(y), weights.data_ptr<float>(), slots.data_ptr<int>(),
                       offsets.data_ptr<int>(), bfm(dy), dw.data_ptr<float>(), (int)T, (int)k, (int)E, (int)D, cur_stream());
  return {dy, dw};
}

void check_group(const Tensor& x, const Tensor& offsets, const char* what) {
  check_rows(x, what);
  check_bf16(x, what);
  TORCH_CHECK(offsets.dim() == 1 && offsets.numel() >= 2, what, ": offsets of at least one expert expected");
  check_ints(offsets, offsets.numel(), x, what);
}

// y[r] = x[r] w[e]^T, or with w_t x[r] w[e]
Tensor do_grouped(const Tensor& x, const Tensor& w, const Tensor& offsets, bool w_t, const Outputs& make) {
  check_group(x, offsets, "grouped_linear");
  check_bf16(w, "grouped_linear: w");
  TORCH_CHECK(w.is_cuda() && w.dim() == 3 && w.is_contiguous() && w.size(0) == offsets.numel() - 1 && w.size(w_t ? 1 : 2) == x.size(1) &&
                  w.device() == x.device(), "grouped_linear: w ", w.sizes(), " does not fit rows of ", x.size(1), " and ",
              offsets.numel() - 1, " experts");
  const int64_t R = x.size(0), K = x.size(1), N = w.size(w_t ? 2 : 1);
  Tensor y = make("grouped_linear", {R, N}, x.options());
  if (R == 0 || N == 0) return y;
  if (K == 0) return y.zero_();
  const int rc = tb::grouped_gemm(bf(x), x.stride(0), bf(w), w_t, offsets.data_ptr<int>(), bfm(y), (int)R, (int)w.size(0), (int)N, (int)K,
                                  attn_err_word().data_ptr<int>(), bind_num_sms(), cur_stream());
  TORCH_CHECK(rc == 0, "grouped_linear failed with code ", rc);
  return y;
}

Tensor do_wgrad(const Tensor& dy, const Tensor& x, const Tensor& offsets, at::ScalarType type, const Outputs& make) {
  check_group(dy, offsets, "grouped_wgrad: dy");
  check_group(x, offsets, "grouped_wgrad: x");
  TORCH_CHECK(dy.size(0) == x.size(0) && dy.device() == x.device(), "grouped_wgrad: ", dy.size(0), " rows and ", x.size(0));
  TORCH_CHECK(type == torch::kBFloat16 || type == torch::kFloat32, "grouped_wgrad: bf16 or fp32 output");
  const int64_t E = offsets.numel() - 1, R = x.size(0), N = dy.size(1), K = x.size(1);
  Tensor dw = make("grouped_wgrad", {E, N, K}, x.options().dtype(type));
  if (N == 0 || K == 0) return dw;
  if (R == 0) return dw.zero_();
  const int rc = tb::grouped_wgrad(bf(dy), dy.stride(0), bf(x), x.stride(0), offsets.data_ptr<int>(), dw.data_ptr(), type == torch::kBFloat16,
                                   (int)R, (int)E, (int)N, (int)K, attn_err_word().data_ptr<int>(), bind_num_sms(), cur_stream());
  TORCH_CHECK(rc == 0, "grouped_wgrad failed with code ", rc);
  return dw;
}

std::tuple<Tensor, Tensor> do_quantize(const Tensor& x) {
  check_rows(x, "quantize8");
  check_bf16(x, "quantize8");
  const int64_t M = x.size(0), N = x.size(1);
  Tensor q = torch::empty({M, N}, x.options().dtype(torch::kInt8));
  Tensor s = torch::empty({M, blocks_of(N)}, x.options().dtype(torch::kFloat32));
  tb::quantize8(bf(x), x.stride(0), q.data_ptr<int8_t>(), s.data_ptr<float>(), M, (int)N, cur_stream());
  return {q, s};
}

void check_kept(const Tensor& q, const Tensor& s, int64_t blocks, const char* what) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 2 && q.is_contiguous() && q.scalar_type() == torch::kInt8 && s.is_cuda() && s.is_contiguous() &&
                  s.scalar_type() == torch::kFloat32 && s.dim() == 2 && s.size(0) == q.size(0) && s.size(1) == blocks &&
                  s.device() == q.device(), what, ": values (int8) and scales (fp32, one for ", tb::kActBlock, " values) do not match");
  TORCH_CHECK(q.size(1) < (1ll << 31), what, ": sizes of 2^31 and more are not supported");
}

Tensor do_dequantize(const Tensor& q, const Tensor& s, const Outputs& make) {
  check_kept(q, s, q.dim() == 2 ? blocks_of(q.size(1)) : 0, "dequantize8");
  Tensor x = make("dequantize8", q.sizes(), q.options().dtype(torch::kBFloat16));
  tb::dequantize8(q.data_ptr<int8_t>(), s.data_ptr<float>(), bfm(x), q.size(0), (int)q.size(1), cur_stream());
  return x;
}

// act, q, scales
std::tuple<Tensor, Tensor, Tensor> do_swiglu8(const Tensor& gu, const Outputs& make) {
  check_rows(gu, "swiglu_8bit");
  check_bf16(gu, "swiglu_8bit");
  TORCH_CHECK(gu.size(1) % 2 == 0, "swiglu_8bit: gate and up columns expected, got an odd number: ", gu.size(1));
  const int64_t M = gu.size(0), F = gu.size(1) / 2;
  Tensor act = make("swiglu_8bit", {M, F}, gu.options());
  Tensor q = torch::empty({M, 2 * F}, gu.options().dtype(torch::kInt8));
  Tensor s = torch::empty({M, 2 * blocks_of(F)}, gu.options().dtype(torch::kFloat32));
  tb::swiglu8_fwd(bf(gu), gu.stride(0), bfm(act), q.data_ptr<int8_t>(), s.data_ptr<float>(), M, (int)F, cur_stream());
  return {act, q, s};
}

Tensor do_swiglu8_bwd(const Tensor& dact, const Tensor& q, const Tensor& s, const Outputs& make) {
  check_rows(dact, "swiglu_8bit backward");
  check_bf16(dact, "swiglu_8bit backward");
  const int64_t M = dact.size(0), F = dact.size(1);
  check_kept(q, s, 2 * blocks_of(F), "swiglu_8bit backward");
  TORCH_CHECK(q.size(0) == M && q.size(1) == 2 * F && q.device() == dact.device(), "swiglu_8bit backward: shapes");
  Tensor dgu = make("swiglu_8bit.bwd", {M, 2 * F}, dact.options());
  tb::swiglu8_bwd(bf(dact), dact.stride(0), q.data_ptr<int8_t>(), s.data_ptr<float>(), bfm(dgu), M, (int)F, cur_stream());
  return dgu;
}

// ---- the whole feed-forward -------------------------------------------------------------------------
void check_experts(const Tensor& x, const Tensor& logits, const Tensor& wgu, const Tensor& wd) {
  check_rows(x, "expert_mlp: x");
  check_bf16(wgu, "expert_mlp: w_gate_up");
  check_bf16(wd, "expert_mlp: w_down");
  const int64_t E = logits.size(1), D = x.size(1);
  TORCH_CHECK(logits.dim() == 2 && logits.size(0) == x.size(0), "expert_mlp: ", x.size(0), " tokens and logits ", logits.sizes());
  TORCH_CHECK(wd.dim() == 3 && wd.size(0) == E && wd.size(1) == D && wd.is_contiguous(), "expert_mlp: w_down ", wd.sizes(),
              " is not [", E, ", ", D, ", units]");
  TORCH_CHECK(wgu.dim() == 3 && wgu.size(0) == E && wgu.size(1) == 2 * wd.size(2) && wgu.size(2) == D && wgu.is_contiguous(),
              "expert_mlp: w_gate_up ", wgu.sizes(), " is not [", E, ", ", 2 * wd.size(2), ", ", D, "]");
  TORCH_CHECK(x.device() == logits.device() && x.device() == wgu.device() && x.device() == wd.device(), "expert_mlp: tensors on several GPUs");
}

// out, aux, weights, experts, slots, offsets, rows, counts, gu (bf16, or q and scales), launches
std::tuple<std::vector<OptTensor>, int64_t> expert_mlp_fwd(const Tensor& x, const Tensor& logits, const Tensor& wgu, const Tensor& wd,
                                                           int64_t k, int64_t capacity, int64_t bits, bool keep,
                                                           const pybind11::object& track) {
  check_experts(x, logits, wgu, wd);
  TORCH_CHECK(bits == 8 || bits == 16, "expert_mlp: activations are kept in 8 or 16 bits, not ", bits);
  const Outputs make{track};
  c10::cuda::CUDAGuard guard(x.device());
  Routed r = do_route(logits, k, capacity, make);
  Tensor xg = do_gather(x, r.rows, k, make);
  Tensor gu = do_grouped(xg, wgu, r.offsets, false, make);
  Tensor act;
  OptTensor q, s;
  if (keep && bits == 8) {
    auto t = do_swiglu8(gu, make);
    act = std::get<0>(t);
    q = std::get<1>(t);
    s = std::get<2>(t);
  } else {
    auto t = do_swiglu8(gu, make);
    act = std::get<0>(t);
  }
  Tensor y = do_grouped(act, wd, r.offsets, false, make);
  Tensor out = do_combine(y, r.weights, r.slots, x.scalar_type(), make);
  OptTensor kept;
  if (keep && bits == 16) kept = gu;
  return {{out, r.aux, r.weights, r.experts, r.slots, r.offsets, r.rows, r.counts, kept, q, s}, 7};
}

// dx, dlogits, dw_gate_up, dw_down, launches
std::tuple<std::vector<OptTensor>, int64_t> expert_mlp_bwd(const Tensor& dout, const OptTensor& daux, const Tensor& x, const Tensor& logits,
                                                           const Tensor& wgu, const Tensor& wd, const Tensor& weights,
                                                           const Tensor& experts, const Tensor& slots, const Tensor& offsets,
                                                           const Tensor& rows, const Tensor& counts, const OptTensor& gu,
                                                           const OptTensor& q, const OptTensor& scales, bool dw_f32,
                                                           const pybind11::object& track) {
  check_experts(x, logits, wgu, wd);
  const Outputs make{track};
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), k = slots.size(1), R = T * k, E = logits.size(1), F = wd.size(2);
  check_ints(slots, R, x, "expert_mlp backward: slots");
  check_ints(offsets, E + 1, x, "expert_mlp backward: offsets");
  TORCH_CHECK(dout.dim() == 2 && dout.size(0) == T && dout.size(1) == x.size(1), "expert_mlp backward: dout");
  if (has(gu)) {
    TORCH_CHECK(gu->is_contiguous() && gu->scalar_type() == torch::kBFloat16 && gu->size(0) == R && gu->size(1) == 2 * F,
                "expert_mlp backward: gu");
  } else {
    TORCH_CHECK(has(q) && has(scales), "expert_mlp backward: no activations were kept");
    check_kept(*q, *scales, 2 * blocks_of(F), "expert_mlp backward");
    TORCH_CHECK(q->size(0) == R && q->size(1) == 2 * F, "expert_mlp backward: kept activations");
  }
  const auto wtype = dw_f32 ? torch::kFloat32 : torch::kBFloat16;
  Tensor dg = do_gather(dout, rows, k, make);
  Tensor s = do_grouped(dg, wd, offsets, true, make);
  Tensor dgu = make("expert_mlp.dgu", {R, 2 * F}, wgu.options());
  Tensor act_w = make("expert_mlp.act", {R, F}, wgu.options());
  Tensor dweights = make("expert_mlp.dweights", {T, k}, weights.options());
  tb::expert_swiglu_bwd(bf(s), has(gu) ? bf(*gu) : nullptr, has(gu) ? nullptr : q->data_ptr<int8_t>(),
                        has(gu) ? nullptr : scales->data_ptr<float>(), weights.data_ptr<float>(), slots.data_ptr<int>(),
                        offsets.data_ptr<int>(), bfm(dgu), bfm(act_w), dweights.data_ptr<float>(), (int)R, (int)E, (int)F, cur_stream());
  Tensor dwd = do_wgrad(dg, act_w, offsets, wtype, make);
  Tensor dxg = do_grouped(dgu, wgu, offsets, true, make);
  Tensor dx = do_combine(dxg, c10::nullopt, slots, x.scalar_type(), make);
  Tensor xg = do_gather(x, rows, k, make);
  Tensor dwgu = do_wgrad(dgu, xg, offsets, wtype, make);
  Tensor dl = do_route_bwd(logits, weights, experts, counts, dweights, daux, make);
  return {{dx, dl, dwgu, dwd}, 9};
}

}  // namespace

void register_moe(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("moe_route", [](const Tensor& logits, int64_t k, int64_t capacity, const py::object& track) {
    c10::cuda::CUDAGuard guard(logits.device());
    Routed r = do_route(logits, k, capacity, Outputs{track});
    return std::make_tuple(r.weights, r.aux, r.experts, r.slots, r.offsets, r.rows, r.counts);
  });
  m.def("moe_route_bwd", [](const Tensor& logits, const Tensor& weights, const Tensor& experts, const Tensor& counts,
                            const OptTensor& dweights, const OptTensor& daux, const py::object& track) {
    c10::cuda::CUDAGuard guard(logits.device());
    return do_route_bwd(logits, weights, experts, counts, dweights, daux, Outputs{track});
  });
  m.def("moe_gather", [](const Tensor& x, const Tensor& rows, int64_t k, const py::object& track) {
    c10::cuda::CUDAGuard guard(x.device());
    return do_gather(x, rows, k, Outputs{track});
  });
  m.def("moe_combine", [](const Tensor& y, const OptTensor& weights, const Tensor& slots, bool f32, const py::object& track) {
    c10::cuda::CUDAGuard guard(y.device());
    return do_combine(y, weights, slots, f32 ? torch::kFloat32 : torch::kBFloat16, Outputs{track});
  });
  m.def("moe_combine_bwd", &combine_bwd);
  m.def("grouped_gemm", [](const Tensor& x, const Tensor& w, const Tensor& offsets, bool w_t, const py::object& track) {
    c10::cuda::CUDAGuard guard(x.device());
    return do_grouped(x, w, offsets, w_t, Outputs{track});
  });
  m.def("grouped_wgrad", [](const Tensor& dy, const Tensor& x, const Tensor& offsets, bool f32, const py::object& track) {
    c10::cuda::CUDAGuard guard(x.device());
    return do_wgrad(dy, x, offsets, f32 ? torch::kFloat32 : torch::kBFloat16, Outputs{track});
  });
  m.def("quantize8", [](const Tensor& x) {
    c10::cuda::CUDAGuard guard(x.device());
    return do_quantize(x);
  });
  m.def("dequantize8", [](const Tensor& q, const Tensor& s, const py::object& track) {
    c10::cuda::CUDAGuard guard(q.device());
    return do_dequantize(q, s, Outputs{track});
  });
  m.def("swiglu8_fwd", [](const Tensor& gu, const py::object& track) {
    c10::cuda::CUDAGuard guard(gu.device());
    return do_swiglu8(gu, Outputs{track});
  });
  m.def("swiglu8_bwd", [](const Tensor& dact, const Tensor& q, const Tensor& s, const py::object& track) {
    c10::cuda::CUDAGuard guard(dact.device());
    return do_swiglu8_bwd(dact, q, s, Outputs{track});
  });
  m.def("expert_mlp_fwd", &expert_mlp_fwd);
  m.def("expert_mlp_bwd", &expert_mlp_bwd);
}
