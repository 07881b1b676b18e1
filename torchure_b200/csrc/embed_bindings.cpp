// Python binding of the embedding lookup, with its autograd node.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>

#include "bind_common.h"
#include "embed_api.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
bool is16(const Tensor& t) { return t.scalar_type() == torch::kBFloat16; }
Tensor rows_of(const Tensor& x) { return x.size(1) <= 1 || x.stride(1) == 1 ? x : x.contiguous(); }

struct Lookup {
  double scale;
  int64_t padding;      // -1: none
  at::ScalarType type;  // of the rows
};

Tensor do_rows(const Tensor& ids, const Tensor& table, const Lookup& how, const Outputs& make) {
  const int64_t T = ids.numel(), V = table.size(0), D = table.size(1);
  auto shape = ids.sizes().vec();
  shape.push_back(D);
  const Tensor out = make("embedding", shape, table.options().dtype(how.type));
  if (T == 0 || D == 0) return out;
  const Tensor rows = rows_of(table);
  const Overlap overlap;
  const int rc = tb::embedding_rows(ids.data_ptr(), ids.scalar_type() == torch::kInt64, rows.data_ptr(), is16(rows), rows.stride(0), out.data_ptr(),
                                    is16(out), (float)how.scale, T, V, (int)D, cur_stream());
  TORCH_CHECK(rc == 0, "embedding failed with code ", rc);
  bind_count_launches(1);
  return out;
}

Tensor do_grad(const Tensor& ids, const Tensor& given, int64_t V, at::ScalarType type, const Lookup& how, const Outputs& make) {
  const int64_t T = ids.numel(), D = given.size(-1);
  const Tensor dtable = make("embedding.dtable", {V, D}, given.options().dtype(type));
  if (D == 0) return dtable;
  if (T == 0) return dtable.zero_();
  const Tensor dout = rows_of(given.reshape({T, D}));
  const Tensor scratch = empty({tb::embedding_scratch_bytes(T, V, (int)D, type == torch::kBFloat16)}, given.options().dtype(torch::kUInt8));
  const Overlap overlap;
  const int rc = tb::embedding_grad(ids.data_ptr(), ids.scalar_type() == torch::kInt64, dout.data_ptr(), is16(dout), dout.stride(0),
                                    dtable.data_ptr(), type == torch::kBFloat16, (float)how.scale, how.padding, T, V, (int)D, scratch.data_ptr(),
                                    cur_stream());
  TORCH_CHECK(rc == 0, "embedding backward failed with code ", rc);
  bind_count_launches(tb::embedding_grad_kernels(T, V, (int)D, type == torch::kBFloat16));
  return dtable;
}

struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, const Lookup& how, bool poison) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["type"] = static_cast<int64_t>(table.scalar_type());
    ctx->saved_data["scale"] = how.scale;
    ctx->saved_data["padding"] = how.padding;
    ctx->saved_data["poison"] = poison;
    return do_rows(ids, table, how, Outputs{poison});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("embedding");
    const Tensor ids = ctx->get_saved_variables()[0];
    c10::cuda::CUDAGuard guard(ids.device());
    const Lookup how{ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), grads[0].scalar_type()};
    return {Tensor(), do_grad(ids, grads[0], ctx->saved_data["rows"].toInt(), static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()), how,
                              Outputs{ctx->saved_data["poison"].toBool()}), Tensor(), Tensor()};
  }
};

Tensor embedding(const Tensor& ids, const Tensor& table, double scale, c10::optional<int64_t> padding, bool out16, bool poison) {
  no_tangents("embedding", table);
  TORCH_CHECK_TYPE(ids.scalar_type() == torch::kInt64 || ids.scalar_type() == torch::kInt32, "embedding: ids in int64 or int32 expected, got ",
                   ids.scalar_type());
  TORCH_CHECK_TYPE(is16(table) || table.scalar_type() == torch::kFloat32, "embedding: a table in bf16 or fp32 expected, got ", table.scalar_type());
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) >= 1, "embedding: a table [rows, width] expected, got ", table.sizes());
  TORCH_CHECK_VALUE(table.is_cuda() && ids.device() == table.device(), "embedding: ids on ", ids.device(), " and a table on ", table.device());
  const int64_t V = table.size(0);
  TORCH_CHECK_VALUE(ids.numel() <= 1ll << 30 && V <= 1ll << 30 && table.size(1) <= 1 << 16, "embedding: ", ids.numel(), " tokens, a table of ",
                    table.sizes(), ": more than 2^30 tokens or rows, or 2^16 columns, are not supported");
  TORCH_CHECK_VALUE(!padding || (*padding >= -V && *padding < V), "embedding: padding_idx ", padding.value_or(0), " in a table of ", V, " rows");
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "embedding: scale ", scale);
  c10::cuda::CUDAGuard guard(table.device());
  const Lookup how{scale, padding ? (*padding < 0 ? *padding + V : *padding) : -1, out16 ? torch::kBFloat16 : torch::kFloat32};
  const Tensor list = ids.contiguous();
  if (!at::GradMode::is_enabled() || !table.requires_grad()) return do_rows(list, table, how, Outputs{poison});
  return EmbeddingNode::apply(list, table, how, poison);
}

}  // namespace

void register_embedding(pybind11::module_& m) { m.def("embedding", &embedding); }
