// Python bindings of the mixture-of-experts kernels and of the 8-bit activation checkpoints, with their autograd nodes: a node in
// Python costs the host 40 - 90 us for a forward and a backward pass, more than most of these kernels run.  Outputs are allocated
// here; in the poison mode (ops/debug.py) each is filled and remembered before its kernel runs.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <atomic>

#include "bind_common.h"
#include "moe_api.h"
#include "pdl.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// torch::empty for GPU tensors without the dispatcher (0.6 us instead of 1.8)
Tensor empty(c10::IntArrayRef size, const at::TensorOptions& options) { return at::detail::empty_cuda(size, options); }

// Backward passes run in threads of autograd's, which do not hold the interpreter's lock.
struct Outputs {
  bool poisoned;
  Tensor operator()(const char* name, c10::IntArrayRef size, const at::TensorOptions& options) const {
    Tensor t = empty(size, options);
    if (poisoned) {
      pybind11::gil_scoped_acquire lock;
      pybind11::module_::import("torchure_b200.ops.debug").attr("track")(name, t);
    }
    return t;
  }
};

// Launches overlap (pdl.h): a kernel comes up while the one before ends, and waits before it reads.  The feed-forward forward, us, without and
// with: 8 experts of 1024 x 1536, 512 rows 48, 39; 4096 rows 83, 70; 32768 rows 284, 278.  (A graph keeps plain edges.)
struct Overlap : tb::PdlScope {
  Overlap() : tb::PdlScope(at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) {}
};

std::atomic<int64_t> g_launches{0};      // kernels launched by the calls of this file

// A launcher's code: counted where it launched, an error otherwise
void done(const char* what, int rc) {
  TORCH_CHECK(rc == 0, what, " failed with code ", rc);
  g_launches += 1;
}

const __nv_bfloat16* bf(const Tensor& t) { return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()); }
__nv_bfloat16* bfm(const Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }
bool at16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

bool bf16_or_f32(const Tensor& t, const char* what) {
  const bool b = t.scalar_type() == torch::kBFloat16;
  TORCH_CHECK_TYPE(b || t.scalar_type() == torch::kFloat32, what, ": bf16 or fp32 expected, got ", t.scalar_type());
  return b;
}
// Indexes of 32 bits in the kernels run past a size by a tile, a block of columns or a grid's stride
constexpr int64_t MAX_SIZE = (1ll << 31) - (1 << 16), MAX_CHOICES = 1 << 30;
void check_size(int64_t n, const char* what) {
  TORCH_CHECK(n <= MAX_SIZE, what, ": sizes of more than 2^31 - 2^16 are not supported, got ", n);
}
// A matrix on the GPU whose rows are contiguous
void check_rows(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), what,
                    ": a matrix on the GPU with contiguous rows expected, got ", t.sizes());
  check_size(t.size(0), what);
  check_size(t.size(1), what);
}
void check_bf16(const Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == torch::kBFloat16, what, ": bf16 expected, got ", t.scalar_type());
}
void check_ints(const Tensor& t, int64_t n, const Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == torch::kInt32 && t.is_contiguous() && t.numel() == n, what, ": contiguous int32 of ", n,
              " elements on the GPU expected");
  TORCH_CHECK_VALUE(t.device() == like.device(), what, ": on another GPU than its operand");
}
int64_t blocks_of(int64_t n) { return (n + tb::kActBlock - 1) / tb::kActBlock; }

struct Routed {
  Tensor weights, experts, slots, offsets, rows, counts, aux;
};

Routed do_route(const Tensor& logits, int64_t k, int64_t capacity, const Outputs& make) {
  check_rows(logits, "route");
  const bool b16 = bf16_or_f32(logits, "route: logits");
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK_VALUE(E >= 1 && E <= tb::kMaxExperts, "route: 1 to ", tb::kMaxExperts, " experts, got ", E);
  TORCH_CHECK_VALUE(k >= 1 && k <= E && k <= tb::kMaxChoices, "route: top_k of ", k, " among ", E, " experts (at most ", tb::kMaxChoices, ")");
  TORCH_CHECK_VALUE(capacity >= 0 && capacity < (1ll << 31), "route: capacity ", capacity);
  TORCH_CHECK_VALUE(T * k <= MAX_CHOICES, "route: too many choices");
  const auto f32 = logits.options().dtype(torch::kFloat32), i32 = logits.options().dtype(torch::kInt32);
  Routed r;
  r.weights = make("route.weights", {T, k}, f32);
  r.aux = make("route.aux", {}, f32);
  r.experts = empty({T, k}, i32);
  r.slots = empty({T, k}, i32);
  r.rows = empty({T * k}, i32);
  if (T == 0) {
    r.offsets = torch::zeros({E + 1}, i32);
    r.counts = torch::zeros({E}, i32);
    r.aux.zero_();
    return r;
  }
  r.offsets = empty({E + 1}, i32);
  r.counts = empty({E}, i32);
  const Tensor scratch = empty({tb::route_scratch_ints((int)T, (int)E, (int)k)}, i32);
  const Overlap overlap;
  const int rc = tb::route_fwd(logits.data_ptr(), b16, logits.stride(0), (int)T, (int)E, (int)k, (int)capacity, r.weights.data_ptr<float>(),
                               r.experts.data_ptr<int>(), r.slots.data_ptr<int>(), r.offsets.data_ptr<int>(), r.rows.data_ptr<int>(),
                               r.counts.data_ptr<int>(), r.aux.data_ptr<float>(), scratch.data_ptr<int>(), cur_stream());
  TORCH_CHECK(rc == 0, "route failed with code ", rc);
  g_launches += tb::route_kernels((int)T, (int)E, (int)k);
  return r;
}

Tensor do_route_bwd(const Tensor& logits, const Tensor& weights, const Tensor& experts, const Tensor& counts, const OptTensor& dweights,
                    const OptTensor& daux, const Outputs& make, Tensor dl = {}) {
  check_rows(logits, "route_bwd");
  const bool b16 = bf16_or_f32(logits, "route_bwd: logits");
  const int64_t T = logits.size(0), E = logits.size(1), k = weights.size(1);
  check_ints(experts, T * k, logits, "route_bwd: experts");
  check_ints(counts, E, logits, "route_bwd: counts");
  TORCH_CHECK(weights.scalar_type() == torch::kFloat32 && weights.is_contiguous() && weights.numel() == T * k, "route_bwd: weights");
  TORCH_CHECK(!has(dweights) || (dweights->scalar_type() == torch::kFloat32 && dweights->is_contiguous() && dweights->numel() == T * k),
              "route_bwd: dweights");
  TORCH_CHECK(!has(daux) || (daux->is_cuda() && daux->scalar_type() == torch::kFloat32 && daux->numel() == 1), "route_bwd: daux");
  if (!dl.defined()) dl = make("route_bwd", {T, E}, logits.options());
  if (T == 0) return dl;
  const Overlap overlap;
  const int rc = tb::route_bwd(logits.data_ptr(), b16, logits.stride(0), weights.data_ptr<float>(), experts.data_ptr<int>(),
                               counts.data_ptr<int>(), has(dweights) ? dweights->data_ptr<float>() : nullptr,
                               has(daux) ? daux->data_ptr<float>() : nullptr, dl.data_ptr(), (int)T, (int)E, (int)k, cur_stream());
  g_launches += 1;
  TORCH_CHECK(rc == 0, "route_bwd failed with code ", rc);
  return dl;
}

// The last argument of the next three: an output that the caller has allocated (on the stream that owns it), or an empty tensor
Tensor do_gather(const Tensor& x, const Tensor& rows, int64_t k, const Outputs& make, Tensor out = {}) {
  check_rows(x, "dispatch");
  const bool b16 = bf16_or_f32(x, "dispatch");
  const int64_t T = x.size(0), D = x.size(1), R = rows.numel();
  check_ints(rows, R, x, "dispatch: rows");
  if (!out.defined()) out = make("dispatch", {R, D}, x.options().dtype(torch::kBFloat16));
  const Overlap overlap;
  done("dispatch",
       tb::rows_gather(x.data_ptr(), b16, x.stride(0), rows.data_ptr<int>(), bfm(out), (int)T, (int)k, (int)R, (int)D, cur_stream()));
  return out;
}

Tensor do_combine(const Tensor& y, const OptTensor& weights, const Tensor& slots, at::ScalarType type, const Outputs& make, Tensor out = {}) {
  check_rows(y, "combine");
  const bool y16 = bf16_or_f32(y, "combine");
  TORCH_CHECK(y.is_contiguous(), "combine: contiguous rows expected");
  const int64_t T = slots.size(0), k = slots.size(1), R = y.size(0), D = y.size(1);
  check_ints(slots, T * k, y, "combine: slots");
  TORCH_CHECK(!has(weights) || (weights->scalar_type() == torch::kFloat32 && weights->is_contiguous() && weights->numel() == T * k &&
                                weights->device() == y.device()), "combine: weights must be contiguous fp32 [tokens, choices]");
  TORCH_CHECK(type == torch::kBFloat16 || type == torch::kFloat32, "combine: bf16 or fp32 output");
  TORCH_CHECK_VALUE(T * ((D + 7) / 8) < (1ll << 31), "combine: 2^34 values and more are not supported");
  if (!out.defined()) out = make("combine", {T, D}, y.options().dtype(type));
  const Overlap overlap;
  done("combine", tb::rows_combine(y.data_ptr(), y16, has(weights) ? weights->data_ptr<float>() : nullptr, slots.data_ptr<int>(),
                                   out.data_ptr(), type == torch::kBFloat16, (int)T, (int)k, (int)R, (int)D, cur_stream()));
  return out;
}

std::tuple<Tensor, Tensor> do_combine_bwd(const Tensor& dout, const Tensor& y, const Tensor& weights, const Tensor& slots,
                                          const Tensor& offsets, const Outputs& make) {
  check_rows(dout, "combine_bwd");
  const bool b16 = bf16_or_f32(dout, "combine_bwd");
  const int64_t T = slots.size(0), k = slots.size(1), D = y.size(1), E = offsets.numel() - 1;
  check_rows(y, "combine_bwd: y");
  check_bf16(y, "combine_bwd: y");
  TORCH_CHECK(y.is_contiguous() && y.size(0) == T * k && dout.size(0) == T && dout.size(1) == D, "combine_bwd: shapes");
  check_ints(slots, T * k, y, "combine_bwd: slots");
  check_ints(offsets, E + 1, y, "combine_bwd: offsets");
  TORCH_CHECK(weights.scalar_type() == torch::kFloat32 && weights.is_contiguous() && weights.numel() == T * k, "combine_bwd: weights");
  Tensor dy = make("combine_bwd.dy", {T * k, D}, y.options());
  Tensor dw = make("combine_bwd.dweights", {T, k}, weights.options());
  if (D == 0 || k == 0) return {dy, dw.zero_()};      // sums of no terms
  const Overlap overlap;
  done("combine backward",
       tb::rows_combine_bwd(dout.data_ptr(), b16, dout.stride(0), bf(y), weights.data_ptr<float>(), slots.data_ptr<int>(),
                            offsets.data_ptr<int>(), bfm(dy), dw.data_ptr<float>(), (int)T, (int)k, (int)E, (int)D, cur_stream()));
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
  TORCH_CHECK_VALUE(offsets.numel() - 1 <= tb::kMaxExperts, "grouped_linear: at most ", tb::kMaxExperts, " experts");
  TORCH_CHECK_VALUE(w.is_cuda() && w.dim() == 3 && w.is_contiguous() && w.size(0) == offsets.numel() - 1 && w.size(w_t ? 1 : 2) == x.size(1) &&
                  w.device() == x.device(), "grouped_linear: w ", w.sizes(), " does not fit rows of ", x.size(1), " and ",
              offsets.numel() - 1, " experts");
  const int64_t R = x.size(0), K = x.size(1), N = w.size(w_t ? 2 : 1);
  Tensor y = make("grouped_linear", {R, N}, x.options());
  if (R == 0 || N == 0) return y;
  if (K == 0) return y.zero_();
  const Overlap overlap;
  const int rc = tb::grouped_gemm(bf(x), x.stride(0), bf(w), w_t, offsets.data_ptr<int>(), bfm(y), (int)R, (int)w.size(0), (int)N, (int)K,
                                  attn_err_word().data_ptr<int>(), bind_num_sms(), cur_stream());
  g_launches += 1;
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
  const Overlap overlap;
  const int rc = tb::grouped_wgrad(bf(dy), dy.stride(0), bf(x), x.stride(0), offsets.data_ptr<int>(), dw.data_ptr(), type == torch::kBFloat16,
                                   (int)R, (int)E, (int)N, (int)K, attn_err_word().data_ptr<int>(), bind_num_sms(), cur_stream());
  g_launches += 1;
  TORCH_CHECK(rc == 0, "grouped_wgrad failed with code ", rc);
  return dw;
}

void check_blocks(int64_t rows, int64_t cols, const char* what) {
  TORCH_CHECK_VALUE(rows * blocks_of(cols) < (1ll << 31), what, ": 2^31 blocks of ", tb::kActBlock, " values and more are not supported");
}

std::tuple<Tensor, Tensor> do_quantize(const Tensor& x) {
  check_rows(x, "quantize8");
  check_bf16(x, "quantize8");
  const int64_t M = x.size(0), N = x.size(1);
  check_blocks(M, N, "quantize8");
  Tensor q = empty({M, N}, x.options().dtype(torch::kInt8));
  Tensor s = empty({M, blocks_of(N)}, x.options().dtype(torch::kFloat32));
  const Overlap overlap;
  done("quantize8", tb::quantize8(bf(x), x.stride(0), q.data_ptr<int8_t>(), s.data_ptr<float>(), M, (int)N, cur_stream()));
  return {q, s};
}

void check_kept(const Tensor& q, const Tensor& s, int64_t blocks, const char* what) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 2 && q.is_contiguous() && q.scalar_type() == torch::kInt8 && s.is_cuda() && s.is_contiguous() &&
                  s.scalar_type() == torch::kFloat32 && s.dim() == 2 && s.size(0) == q.size(0) && s.size(1) == blocks &&
                  s.device() == q.device(), what, ": values (int8) and scales (fp32, one for ", tb::kActBlock, " values) do not match");
  check_size(q.size(1), what);
}

Tensor do_dequantize(const Tensor& q, const Tensor& s, const Outputs& make) {
  check_kept(q, s, q.dim() == 2 ? blocks_of(q.size(1)) : 0, "dequantize8");
  check_blocks(q.size(0), q.size(1), "dequantize8");
  Tensor x = make("dequantize8", q.sizes(), q.options().dtype(torch::kBFloat16));
  const Overlap overlap;
  done("dequantize8", tb::dequantize8(q.data_ptr<int8_t>(), s.data_ptr<float>(), bfm(x), q.size(0), (int)q.size(1), cur_stream()));
  return x;
}

// act, and with `keep` q and scales
std::tuple<Tensor, Tensor, Tensor> do_swiglu8(const Tensor& gu, bool keep, const Outputs& make) {
  check_rows(gu, "swiglu_8bit");
  check_bf16(gu, "swiglu_8bit");
  TORCH_CHECK(gu.size(1) % 2 == 0, "swiglu_8bit: gate and up columns expected, got an odd number: ", gu.size(1));
  const int64_t M = gu.size(0), F = gu.size(1) / 2;
  check_blocks(M, F, "swiglu_8bit");
  Tensor act = make("swiglu_8bit", {M, F}, gu.options());
  Tensor q, s;
  if (keep) {
    q = empty({M, 2 * F}, gu.options().dtype(torch::kInt8));
    s = empty({M, 2 * blocks_of(F)}, gu.options().dtype(torch::kFloat32));
  }
  const Overlap overlap;
  done("swiglu_8bit", tb::swiglu8_fwd(bf(gu), gu.stride(0), bfm(act), keep ? q.data_ptr<int8_t>() : nullptr,
                                      keep ? s.data_ptr<float>() : nullptr, M, (int)F, cur_stream()));
  return {act, q, s};
}

Tensor do_swiglu8_bwd(const Tensor& dact, const Tensor& q, const Tensor& s, const Outputs& make) {
  check_rows(dact, "swiglu_8bit backward");
  check_bf16(dact, "swiglu_8bit backward");
  const int64_t M = dact.size(0), F = dact.size(1);
  check_kept(q, s, 2 * blocks_of(F), "swiglu_8bit backward");
  TORCH_CHECK(q.size(0) == M && q.size(1) == 2 * F && q.device() == dact.device(), "swiglu_8bit backward: shapes");
  Tensor dgu = make("swiglu_8bit.bwd", {M, 2 * F}, dact.options());
  const Overlap overlap;
  done("swiglu_8bit backward",
       tb::swiglu8_bwd(bf(dact), dact.stride(0), q.data_ptr<int8_t>(), s.data_ptr<float>(), bfm(dgu), M, (int)F, cur_stream()));
  return dgu;
}

// ---- operands as the kernels read them ---------------------------------------------------------------
// x with contiguous rows (a copy only where it has none)
Tensor rows_of(const Tensor& x) { return x.size(-1) <= 1 || x.stride(-1) == 1 ? x : x.contiguous(); }
// x [R, K] with columns in eights (zeros behind), the row stride and the base on 16 bytes
Tensor operand(const Tensor& x) {
  if (x.size(1) % 8 == 0 && x.stride(1) == 1 && x.stride(0) % 8 == 0 && x.stride(0) >= x.size(1) && at16(x))
    return x;
  return x.size(1) % 8 ? at::constant_pad_nd(x, {0, (8 - x.size(1) % 8) % 8}).contiguous() : x.clone(at::MemoryFormat::Contiguous);
}
// w [E, N, K] in bf16, both widths in eights (zeros behind)
Tensor matrices(const Tensor& w) {
  Tensor b = w.scalar_type() == torch::kBFloat16 ? w : w.to(torch::kBFloat16);
  const int64_t n = (8 - w.size(1) % 8) % 8, k = (8 - w.size(2) % 8) % 8;
  b = n || k ? at::constant_pad_nd(b, {0, k, 0, n}).contiguous() : b.contiguous();
  return at16(b) ? b : b.clone();
}

// ---- autograd nodes ----------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void only_once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient itself has no gradient (create_graph is not supported)");
}
// A dual tensor asks for no gradient, so that calls without gradients would pass its tangent by
template <class... Ts>
void no_tangents(const char* what, const Ts&... tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(... || (tensors.defined() && tensors._fw_grad(0).defined())), what,
                              ": forward-mode derivatives are not supported");
}
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

struct RouteNode : torch::autograd::Function<RouteNode> {
  // weights, aux, experts, slots, offsets, rows, counts
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k, int64_t capacity, bool poison) {
    Routed r = do_route(logits, k, capacity, Outputs{poison});
    ctx->save_for_backward({logits, r.weights, r.experts, r.counts});
    ctx->saved_data["poison"] = poison;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r.experts, r.slots, r.offsets, r.rows, r.counts});
    return {r.weights, r.aux, r.experts, r.slots, r.offsets, r.rows, r.counts};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("route");
    const auto s = ctx->get_saved_variables();
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    c10::cuda::CUDAGuard guard(s[0].device());
    const Tensor dw = grads[0].defined() ? grads[0].to(torch::kFloat32).contiguous() : grads[0];
    const Tensor da = grads[1].defined() ? grads[1].to(torch::kFloat32) : grads[1];
    return {do_route_bwd(s[0], s[1], s[2], s[3], opt(dw), opt(da), Outputs{ctx->saved_data["poison"].toBool()}), Tensor(), Tensor(), Tensor()};
  }
};

// Logits as the kernels read them: fp32 or bf16, others in fp32
Tensor router_logits(const Tensor& t) {
  return !t.is_floating_point() || t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16 ? t : t.to(torch::kFloat32);
}

variable_list moe_route(const Tensor& logits, int64_t k, int64_t capacity, bool poison) {
  no_tangents("route", logits);
  TORCH_CHECK_VALUE(logits.dim() == 2 && logits.is_floating_point(), "route: logits [tokens, experts] expected, got ", logits.scalar_type(),
                    " ", logits.sizes());
  c10::cuda::CUDAGuard guard(logits.device());
  const Tensor rows = rows_of(router_logits(logits));
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
    Routed r = do_route(rows, k, capacity, Outputs{poison});
    return {r.weights, r.aux, r.experts, r.slots, r.offsets, r.rows, r.counts};
  }
  return RouteNode::apply(rows, k, capacity, poison);
}

struct DispatchNode : torch::autograd::Function<DispatchNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& slots, const Tensor& rows, bool poison) {
    ctx->save_for_backward({slots});
    ctx->saved_data["type"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["poison"] = poison;
    return do_gather(x, rows, slots.size(1), Outputs{poison});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("dispatch");
    const Tensor slots = ctx->get_saved_variables()[0];
    c10::cuda::CUDAGuard guard(slots.device());
    return {do_combine(grads[0].contiguous(), c10::nullopt, slots, static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()),
                       Outputs{ctx->saved_data["poison"].toBool()}), Tensor(), Tensor(), Tensor()};
  }
};

Tensor moe_dispatch(const Tensor& x, const Tensor& slots, const Tensor& rows, bool poison) {
  no_tangents("dispatch", x);
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK_VALUE(x.dim() == 2 && slots.dim() == 2 && x.size(0) == slots.size(0), "dispatch: ", slots.size(0), " tokens were routed, got ",
                    x.sizes());
  TORCH_CHECK_VALUE(rows.numel() <= MAX_CHOICES, "dispatch: too many choices");
  check_ints(slots, rows.numel(), x, "dispatch: slots");
  return DispatchNode::apply(rows_of(x), slots, rows, poison);
}

struct CombineNode : torch::autograd::Function<CombineNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const Tensor& slots, const Tensor& offsets, bool f32,
                        bool poison) {
    ctx->save_for_backward({y, weights, slots, offsets});
    ctx->saved_data["poison"] = poison;
    return do_combine(y, weights, slots, f32 ? torch::kFloat32 : torch::kBFloat16, Outputs{poison});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("combine");
    const auto s = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(s[0].device());
    auto r = do_combine_bwd(rows_of(grads[0]), s[0], s[1], s[2], s[3], Outputs{ctx->saved_data["poison"].toBool()});
    return {std::get<0>(r), std::get<1>(r), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor moe_combine(const Tensor& y, const Tensor& weights, const Tensor& slots, const Tensor& offsets, bool f32, bool poison) {
  no_tangents("combine", y, weights);
  check_bf16(y, "combine");
  c10::cuda::CUDAGuard guard(y.device());
  TORCH_CHECK_VALUE(y.dim() == 2 && slots.dim() == 2 && y.size(0) == slots.numel(), "combine: ", slots.numel(), " rows expected, got ",
                    y.sizes());
  TORCH_CHECK_VALUE(slots.numel() <= MAX_CHOICES, "combine: too many choices");
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() >= 2, "combine: offsets of at least one expert expected, got ", offsets.sizes());
  check_ints(offsets, offsets.numel(), y, "combine: offsets");
  return CombineNode::apply(y.contiguous(), weights.contiguous(), slots, offsets, f32, poison);
}

struct GroupedNode : torch::autograd::Function<GroupedNode> {
  // with columns in eights, as the kernel writes them
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& offsets, bool poison) {
    const Tensor xb = operand(x), wb = matrices(w);
    const Tensor y = do_grouped(xb, wb, offsets, false, Outputs{poison});
    ctx->save_for_backward({xb, wb, offsets});
    ctx->saved_data["n"] = w.size(1);
    ctx->saved_data["k"] = w.size(2);
    ctx->saved_data["type"] = static_cast<int64_t>(w.scalar_type());
    ctx->saved_data["poison"] = poison;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("grouped_linear");
    const auto s = ctx->get_saved_variables();
    const int64_t n = ctx->saved_data["n"].toInt(), k = ctx->saved_data["k"].toInt();
    const Outputs make{ctx->saved_data["poison"].toBool()};
    c10::cuda::CUDAGuard guard(s[0].device());
    const Tensor dy = operand(grads[0]);
    Tensor dx, dw;
    if (ctx->needs_input_grad(0)) {
      dx = do_grouped(dy, s[1], s[2], true, make);
      if (dx.size(1) != k) dx = dx.narrow(1, 0, k);
    }
    if (ctx->needs_input_grad(1)) {
      dw = do_wgrad(dy, s[0], s[2], static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()), make);
      if (dw.size(1) != n || dw.size(2) != k) dw = dw.narrow(1, 0, n).narrow(2, 0, k);
    }
    return {dx, dw, Tensor(), Tensor()};
  }
};

Tensor grouped_linear(const Tensor& x, const Tensor& w, const Tensor& offsets, bool poison) {
  no_tangents("grouped_linear", x, w);
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 3 && x.size(1) == w.size(2), "grouped_linear: rows ", x.sizes(), " and matrices ", w.sizes(),
                    " do not fit");
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() == w.size(0) + 1, "grouped_linear: ", w.size(0) + 1, " offsets expected, got ",
                    offsets.sizes());
  TORCH_CHECK_TYPE(x.scalar_type() == torch::kBFloat16 && (w.scalar_type() == torch::kBFloat16 || w.scalar_type() == torch::kFloat32),
                   "grouped_linear: bf16 rows and bf16 or fp32 matrices expected, got ", x.scalar_type(), " and ", w.scalar_type());
  TORCH_CHECK_VALUE(offsets.scalar_type() == torch::kInt32 && offsets.device() == x.device() && w.device() == x.device(),
                    "grouped_linear: int32 offsets and matrices on the GPU of the rows expected");
  for (const int64_t n : {x.size(0), x.size(1), w.size(1)}) check_size(n, "grouped_linear");
  c10::cuda::CUDAGuard guard(x.device());
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || w.requires_grad())) {
    const Tensor y = do_grouped(operand(x), matrices(w), offsets.contiguous(), false, Outputs{poison});
    return y.size(1) == w.size(1) ? y : y.narrow(1, 0, w.size(1)).detach();
  }
  // (a view made inside the node, or without gradients and not detached, could not be changed in place)
  const Tensor y = GroupedNode::apply(x, w, offsets.contiguous(), poison);
  return y.size(1) == w.size(1) ? y : y.narrow(1, 0, w.size(1));
}

struct Swiglu8Node : torch::autograd::Function<Swiglu8Node> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gu, bool poison) {
    auto r = do_swiglu8(gu, true, Outputs{poison});
    ctx->save_for_backward({std::get<1>(r), std::get<2>(r)});
    ctx->saved_data["poison"] = poison;
    return std::get<0>(r);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("swiglu_8bit");
    const auto s = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(s[0].device());
    return {do_swiglu8_bwd(rows_of(grads[0]), s[0], s[1], Outputs{ctx->saved_data["poison"].toBool()}), Tensor()};
  }
};

Tensor swiglu_8bit(const Tensor& gu, bool poison) {
  no_tangents("swiglu_8bit", gu);
  check_bf16(gu, "swiglu_8bit");
  TORCH_CHECK_VALUE(gu.dim() >= 1 && gu.size(-1) % 2 == 0, "swiglu_8bit: gate and up columns expected, got ", gu.sizes());
  c10::cuda::CUDAGuard guard(gu.device());
  auto shape = gu.sizes().vec();
  const Tensor rows = rows_of(gu.dim() == 2 ? gu : gu.reshape({-1, shape.back()}));
  const bool keep = at::GradMode::is_enabled() && gu.requires_grad();
  const Tensor act = keep ? Swiglu8Node::apply(rows, poison) : std::get<0>(do_swiglu8(rows, false, Outputs{poison}));
  shape.back() /= 2;
  return gu.dim() == 2 ? act : act.view(shape);
}

// ---- the whole feed-forward -------------------------------------------------------------------------
struct Mlp {
  Tensor out;
  Routed r;
  Tensor gu, q, scales;      // what the backward pass reads: gate | up in bf16, or in 8 bits
};

// A pass without gradients of up to four tokens runs in the two kernels of moe_token.cu, which read an expert once for every token that
// chose it, unless that is more than 80 MB: the general path reads it once.  Measured on B200, us, general path, token kernels: experts x
// choices x width x units 8 x 2 x 1024 x 1536, one token 36, 17, four (75 MB) 30, 24; 64 x 4 x 1024 x 768, four (75 MB) 30, 26; 64 x 8 x
// 2048 x 1024, one (100 MB) 38, 43, two 53, 57, four 71, 107.
constexpr int64_t TOKEN_MAX = 4, TOKEN_BYTES = 80 << 20;
// From here on the backward pass runs gather, sum and the router's gradient beside the products: a training pass over 4096 rows (8 experts of
// 1024 x 1536) takes 227 us instead of 231, over 8192 294 instead of 299; the events cost the host 5 us, which has the last word below.
constexpr int64_t BESIDE_MIN_ROWS = 4096;

bool runs_by_token(const Tensor& x, int64_t k, const Tensor& wgu, const Tensor& wd) {
  return x.size(0) >= 1 && x.size(0) <= TOKEN_MAX && x.size(0) * k <= tb::kTokenChoices && x.stride(0) % 8 == 0 &&
         x.size(0) * k * wd.size(1) * wd.size(2) * 6 <= TOKEN_BYTES &&
         at16(x) && at16(wgu) && at16(wd);
}

// out, aux
variable_list mlp_by_token(const Tensor& x, const Tensor& logits, const Tensor& wgu, const Tensor& wd, int64_t k, int64_t capacity,
                           const Outputs& make) {
  const int64_t T = x.size(0), D = x.size(1), E = wd.size(0), F = wd.size(2);
  TORCH_CHECK_VALUE(E <= tb::kMaxExperts, "expert_mlp: 1 to ", tb::kMaxExperts, " experts, got ", E);
  TORCH_CHECK_VALUE(k >= 1 && k <= E && k <= tb::kMaxChoices, "expert_mlp: top_k of ", k, " among ", E, " experts (at most ",
                    tb::kMaxChoices, ")");
  TORCH_CHECK_VALUE(capacity >= 0 && capacity < (1ll << 31), "expert_mlp: capacity ", capacity);
  const Tensor out = make("expert_mlp.out", {T, D}, x.options()), aux = make("expert_mlp.aux", {}, x.options().dtype(torch::kFloat32));
  const Tensor scratch = empty({tb::token_scratch_bytes((int)T, (int)k, (int)F)}, x.options().dtype(torch::kUInt8));
  const int rc = tb::token_mlp(logits.data_ptr(), bf16_or_f32(logits, "expert_mlp: logits"), logits.stride(0), x.data_ptr(),
                               x.scalar_type() == torch::kBFloat16, x.stride(0), bf(wgu), bf(wd), out.data_ptr(), aux.data_ptr<float>(),
                               scratch.data_ptr(), (int)T, (int)E, (int)k, (int)capacity, (int)D, (int)F, cur_stream());
  TORCH_CHECK(rc == 0, "expert_mlp failed with code ", rc);
  g_launches += 2;
  return {out, aux};
}

// Whether the gate / up product reads token rows where they lie: few rows per expert, bf16, on 16 bytes.  Others are put in expert order
// first, rounded where they are fp32.
bool rows_stay(const Tensor& x, int64_t R, int64_t E, bool in8) {
  return tb::grouped_swiglu_listed((int)R, (int)E) && !in8 && x.scalar_type() == torch::kBFloat16 && x.stride(1) == 1 &&
         x.stride(0) % 8 == 0 && x.stride(0) >= x.size(1) && at16(x);
}

// Rounded to bf16 between the kernels are gate and up (kept for the backward pass only), the activation (the down product's operand) and, unless
// rows are few, the down product's rows, which the weighted sum reads back: in fp32 they would be 67 MB more of traffic (16384 rows of 1024).
// Weights, sums and the weighted sum are fp32.
Mlp mlp_fwd(const Tensor& x, const Tensor& logits, const Tensor& wgu, const Tensor& wd, int64_t k, int64_t capacity, int64_t bits, bool keep,
            const Outputs& make) {
  Mlp m;
  const Overlap overlap;
  m.r = do_route(logits, k, capacity, make);
  const int64_t R = x.size(0) * k, F = wd.size(2), E = wd.size(0), D = x.size(1);
  const Tensor act = make("expert_mlp.act", {R, F}, wgu.options());
  if (keep && bits == 16) m.gu = make("expert_mlp.gu", {R, 2 * F}, wgu.options());
  if (keep && bits == 8) {
    m.q = empty({R, 2 * F}, wgu.options().dtype(torch::kInt8));
    m.scales = make("expert_mlp.scales", {R, 2 * blocks_of(F)}, wgu.options().dtype(torch::kFloat32));
  }
  if (R > 0) {
    const bool listed = rows_stay(x, R, E, m.q.defined());
    const Tensor xg = listed ? x : do_gather(x, m.r.rows, k, make);
    const int rc = tb::grouped_swiglu(
        bf(xg), xg.stride(0), listed ? m.r.rows.data_ptr<int>() : nullptr, (int)k, (int)x.size(0), bf(wgu), m.r.offsets.data_ptr<int>(),
        bfm(act), m.gu.defined() ? bfm(m.gu) : nullptr, m.q.defined() ? m.q.data_ptr<int8_t>() : nullptr,
        m.q.defined() ? m.scales.data_ptr<float>() : nullptr, (int)R, (int)E, (int)F, (int)D, true, attn_err_word().data_ptr<int>(),
        bind_num_sms(), cur_stream());
    TORCH_CHECK(rc == 0, "expert_mlp: gate / up product failed with code ", rc);
    g_launches += 1;
  }
  Tensor y;
  if (R > 0 && tb::grouped_gemm_few((int)R, (int)E)) {
    y = make("expert_mlp.y", {R, D}, wgu.options().dtype(torch::kFloat32));
    const int rc = tb::grouped_gemm_f32(bf(act), F, bf(wd), m.r.offsets.data_ptr<int>(), y.data_ptr<float>(), (int)R, (int)E, (int)D, (int)F,
                                        true, attn_err_word().data_ptr<int>(), bind_num_sms(), cur_stream());
    TORCH_CHECK(rc == 0, "expert_mlp: down product failed with code ", rc);
    g_launches += 1;
  } else {
    y = do_grouped(act, wd, m.r.offsets, false, make);
  }
  m.out = do_combine(y, m.r.weights, m.r.slots, x.scalar_type(), make);
  return m;
}

// A second stream for row kernels that have nothing to do with the product on the current one: they are bound by memory and fit beside its
// CTAs.  What they read and write is allocated on the current stream before and outlives this object, and the current stream waits for the
// second one before it goes: to the allocator there is one stream.
class Beside {
 public:
  explicit Beside(bool on) : main_(at::cuda::getCurrentCUDAStream()), on_(on) {
    if (on_) side_ = at::cuda::getStreamFromPool(false, main_.device_index());
  }
  // runs f on the second stream, behind everything on the current one so far
  template <class F>
  void run(F f) {
    if (!on_) return f();
    from_.record(main_);
    from_.block(*side_);
    c10::cuda::CUDAStreamGuard guard(*side_);
    f();
    busy_ = true;
  }
  // the current stream waits for what was run
  void join() {
    if (!busy_) return;
    back_.record(*side_);
    back_.block(main_);
    busy_ = false;
  }
  ~Beside() {
    try {
      join();
    } catch (...) {      // (behind an error that is on its way already)
    }
  }

 private:
  c10::cuda::CUDAStream main_;
  c10::optional<c10::cuda::CUDAStream> side_;
  at::cuda::CUDAEvent from_, back_;
  bool on_, busy_ = false;
};

struct Wanted {
  bool x, logits, gate_up, down;
};

// dx, dlogits, dw_gate_up, dw_down, undefined where not wanted
variable_list mlp_bwd(const Tensor& dout, const OptTensor& daux, const Tensor& x, const Tensor& logits, const Tensor& wgu, const Tensor& wd,
                      const Routed& r, const Tensor& gu, const Tensor& q, const Tensor& scales, at::ScalarType wtype, const Wanted& wanted,
                      const Outputs& make) {
  const int64_t T = x.size(0), k = r.slots.size(1), R = T * k, E = logits.size(1), F = wd.size(2);
  if (R == 0)
    return {at::zeros_like(x), at::zeros_like(logits), at::zeros(wgu.sizes(), wgu.options().dtype(wtype)),
            at::zeros(wd.sizes(), wd.options().dtype(wtype))};
  Tensor dgu = make("expert_mlp.dgu", {R, 2 * F}, wgu.options());
  Tensor act_w = make("expert_mlp.act", {R, F}, wgu.options());
  Tensor dweights = make("expert_mlp.dweights", {T, k}, r.weights.options());
  Tensor dg, s, dxg, dwd, dwgu, xg, dx, dl;
  if (wanted.gate_up) xg = make("expert_mlp.xg", {R, x.size(1)}, wgu.options());
  if (wanted.x) dx = make("expert_mlp.dx", {T, x.size(1)}, x.options());
  if (wanted.logits) dl = make("expert_mlp.dlogits", {T, E}, logits.options());
  const Overlap overlap;
  Beside beside(R >= BESIDE_MIN_ROWS);
  dg = do_gather(dout, r.rows, k, make);
  if (wanted.gate_up) beside.run([&] { do_gather(x, r.rows, k, make, xg); });
  s = do_grouped(dg, wd, r.offsets, true, make);
  const bool kept16 = gu.defined();
  done("expert_mlp backward",
       tb::expert_swiglu_bwd(bf(s), kept16 ? bf(gu) : nullptr, kept16 ? nullptr : q.data_ptr<int8_t>(),
                             kept16 ? nullptr : scales.data_ptr<float>(), r.weights.data_ptr<float>(), r.slots.data_ptr<int>(),
                             r.offsets.data_ptr<int>(), bfm(dgu), bfm(act_w), dweights.data_ptr<float>(), (int)R, (int)E, (int)F, cur_stream()));
  if (wanted.x) dxg = do_grouped(dgu, wgu, r.offsets, true, make);
  if (wanted.x || wanted.logits)
    beside.run([&] {
      if (wanted.x) do_combine(dxg, c10::nullopt, r.slots, x.scalar_type(), make, dx);
      if (wanted.logits) do_route_bwd(logits, r.weights, r.experts, r.counts, dweights, daux, make, dl);
    });
  if (wanted.down) dwd = do_wgrad(dg, act_w, r.offsets, wtype, make);
  beside.join();
  if (wanted.gate_up) dwgu = do_wgrad(dgu, xg, r.offsets, wtype, make);
  return {dx, dl, dwgu, dwd};
}

// gate and up matrices as one bf16 stack [E, 2F, D]: given as one, or as a pair
Tensor stack_of(const Tensor& first, const OptTensor& second) {
  if (!has(second)) return matrices(first);
  const int64_t E = first.size(0), F = first.size(1), D = first.size(2);
  Tensor w = empty({E, 2 * F, D}, first.options().dtype(torch::kBFloat16));
  w.narrow(1, 0, F).copy_(first);
  w.narrow(1, F, F).copy_(*second);
  return w;
}

struct MlpNode : torch::autograd::Function<MlpNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& logits, const Tensor& first, const OptTensor& second,
                               const Tensor& wd, int64_t k, int64_t capacity, int64_t bits, bool poison) {
    const Tensor wgu = stack_of(first, second), wdb = matrices(wd);
    Mlp m = mlp_fwd(x, logits, wgu, wdb, k, capacity, bits, true, Outputs{poison});
    ctx->save_for_backward({x, logits, wgu, wdb, m.r.weights, m.r.experts, m.r.slots, m.r.offsets, m.r.rows, m.r.counts, m.gu, m.q, m.scales});
    ctx->saved_data["type"] = static_cast<int64_t>(wd.scalar_type());
    ctx->saved_data["pair"] = has(second);
    ctx->saved_data["poison"] = poison;
    ctx->set_materialize_grads(false);
    return {m.out, m.r.aux};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("expert_mlp");
    const auto s = ctx->get_saved_variables();
    const Outputs make{ctx->saved_data["poison"].toBool()};
    variable_list out(9);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    c10::cuda::CUDAGuard guard(s[0].device());
    const Tensor daux = grads[1].defined() ? grads[1].to(torch::kFloat32) : grads[1];
    if (!grads[0].defined()) {
      out[1] = do_route_bwd(s[1], s[4], s[5], s[9], c10::nullopt, opt(daux), make);
      return out;
    }
    Routed r{s[4], s[5], s[6], s[7], s[8], s[9], Tensor()};
    // edges are those of the tensors that were given: x, logits, gate (and up), down
    const bool pair = ctx->saved_data["pair"].toBool();
    const Wanted wanted{ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2) || (pair && ctx->needs_input_grad(3)),
                        ctx->needs_input_grad(pair ? 4 : 3)};
    auto g = mlp_bwd(rows_of(grads[0]), opt(daux), s[0], s[1], s[2], s[3], r, s[10], s[11], s[12],
                     static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()), wanted, make);
    const int64_t F = s[3].size(2);
    out[0] = g[0];
    out[1] = g[1];
    if (wanted.gate_up) out[2] = pair ? g[2].narrow(1, 0, F) : g[2];
    if (wanted.gate_up && pair) out[3] = g[2].narrow(1, F, F);
    out[4] = g[3];
    return out;
  }
};

variable_list expert_mlp(const Tensor& x, const Tensor& given_logits, const Tensor& first, const OptTensor& second, const Tensor& wd, int64_t k,
                         int64_t capacity, int64_t bits, bool poison) {
  no_tangents("expert_mlp", x, given_logits, first, has(second) ? *second : Tensor(), wd);
  check_rows(x, "expert_mlp: x");
  check_rows(given_logits, "expert_mlp: logits");
  const Tensor logits = router_logits(given_logits);
  bf16_or_f32(x, "expert_mlp: x");
  bf16_or_f32(first, "expert_mlp: w_gate_up");
  TORCH_CHECK_TYPE(first.scalar_type() == wd.scalar_type(), "expert_mlp: matrices of one type expected, got ", first.scalar_type(), " and ",
                   wd.scalar_type());
  TORCH_CHECK_VALUE(bits == 8 || bits == 16, "expert_mlp: activations are kept in 8 or 16 bits, not ", bits);
  const bool pair = has(second);
  TORCH_CHECK_VALUE(!pair || (second->sizes() == first.sizes() && second->scalar_type() == first.scalar_type() &&
                              second->device() == first.device()),
                    "expert_mlp: w_gate and w_up differ");
  TORCH_CHECK_VALUE(wd.dim() == 3 && first.dim() == 3, "expert_mlp: matrices [E, 2F, D] and [E, D, F] expected");
  const int64_t E = wd.size(0), D = wd.size(1), F = wd.size(2);
  TORCH_CHECK_VALUE(first.size(0) == E && first.size(1) == (pair ? F : 2 * F) && first.size(2) == D && x.size(1) == D &&
                        logits.size(0) == x.size(0) && logits.size(1) == E, "expert_mlp: x ", x.sizes(), ", logits ", logits.sizes(),
                    ", w_gate_up ", first.sizes(), ", w_down ", wd.sizes(), " do not fit");
  TORCH_CHECK_VALUE(D % 8 == 0 && F % 8 == 0 && D > 0 && F > 0, "expert_mlp: widths in multiples of 8 expected, got D ", D, " and F ", F);
  check_size(D, "expert_mlp");
  check_size(2 * F, "expert_mlp");
  TORCH_CHECK_VALUE(x.device() == logits.device() && x.device() == first.device() && x.device() == wd.device(),
                    "expert_mlp: tensors on several GPUs");
  c10::cuda::CUDAGuard guard(x.device());
  const bool keep = at::GradMode::is_enabled() &&
                    (x.requires_grad() || logits.requires_grad() || first.requires_grad() || wd.requires_grad() ||
                     (pair && second->requires_grad()));
  if (keep) return MlpNode::apply(x, logits, first, second, wd, k, capacity, bits, poison);
  const Tensor wgu = stack_of(first, second), wdb = matrices(wd);
  if (runs_by_token(x, k, wgu, wdb)) {
    const Overlap overlap;
    return mlp_by_token(x, logits, wgu, wdb, k, capacity, Outputs{poison});
  }
  Mlp m = mlp_fwd(x, logits, wgu, wdb, k, capacity, bits, false, Outputs{poison});
  return {m.out, m.r.aux};
}

}  // namespace

void register_moe(pybind11::module_& m) {
  m.def("moe_route", &moe_route, "(weights, aux, experts, slots, offsets, rows, counts)");
  m.def("moe_dispatch", &moe_dispatch);
  m.def("moe_combine", &moe_combine);
  m.def("grouped_linear", &grouped_linear);
  m.def("expert_mlp", &expert_mlp, "(out, aux)");
  m.def("quantize8", [](const Tensor& x) {
    TORCH_CHECK_VALUE(x.dim() == 2, "quantize8: a matrix expected, got ", x.dim(), " dimensions");
    c10::cuda::CUDAGuard guard(x.device());
    return do_quantize(rows_of(x));
  });
  m.def("dequantize8", [](const Tensor& q, const Tensor& s, bool poison) {
    TORCH_CHECK_VALUE(q.is_cuda(), "dequantize8: a tensor on the GPU expected");
    c10::cuda::CUDAGuard guard(q.device());
    return do_dequantize(q, s, Outputs{poison});
  });
  m.def("swiglu_8bit", &swiglu_8bit);
  m.def("moe_launches", [](bool reset) { return reset ? g_launches.exchange(0) : g_launches.load(); },
        "kernels launched by the operators of this file since the last reset");
}
