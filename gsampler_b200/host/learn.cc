#include "learn.h"

#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>

#include <atomic>
#include <cmath>
#include <mutex>

#include "graph.h"
#include "gsb200.h"

namespace gsb_host {

static int ValueType(const torch::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.defined(), op, ": ", name, " is undefined");
  TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor (this library has no CPU path)");
  switch (t.scalar_type()) {
    case torch::kFloat32: return GSB_F32;
    case torch::kFloat16: return GSB_F16;
    case torch::kBFloat16: return GSB_BF16;
    default: TORCH_CHECK(false, op, ": ", name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  }
}

static void CheckIndex(const torch::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.defined() && t.is_cuda(), op, ": ", name, " must be a CUDA tensor (this library has no CPU path)");
  TORCH_CHECK(t.scalar_type() == torch::kInt64, op, ": ", name, " must be int64");
}

static void CheckScale(double scale, const char* op) {
  TORCH_CHECK(std::isfinite((float)scale), op, ": scale must be finite as a float32, got ", scale);
}

static int* ErrorWord(const torch::Device& dev) { return AsyncErrorWord(dev).data_ptr<int>(); }

// ------------------------------------------------------------------ embedding
torch::Tensor Embedding(torch::Tensor weight, torch::Tensor index, double scale, int64_t padding) {
  const int dt = ValueType(weight, "Embedding", "weight");
  CheckIndex(index, "Embedding", "index");
  TORCH_CHECK(weight.device() == index.device(), "Embedding: weight and index live on different devices");
  TORCH_CHECK(weight.dim() == 2, "Embedding: weight must be two-dimensional");
  CheckScale(scale, "Embedding");
  c10::cuda::CUDAGuard guard(index.device());
  // rows may be strided (a column slice of a wider table is read in place)
  if (weight.size(1) > 1 && weight.stride(1) != 1) weight = weight.contiguous();
  if (weight.size(0) > 1 && weight.stride(0) < weight.size(1)) weight = weight.contiguous();
  index = index.contiguous();
  auto sizes = index.sizes().vec();
  sizes.push_back(weight.size(1));
  auto out = torch::empty(sizes, weight.options());
  const int64_t ld = weight.size(0) > 1 ? weight.stride(0) : weight.size(1);
  CheckStatus(gsb_embedding(weight.data_ptr(), dt, ld, weight.size(0), weight.size(1), index.data_ptr<int64_t>(),
                            index.numel(), (float)scale, padding, out.data_ptr(), ErrorWord(index.device()),
                            CurrentStream()),
              "embedding");
  return out;
}

static void CheckEmbeddingGrad(const torch::Tensor& grad, const torch::Tensor& index, int64_t num_rows, double scale) {
  CheckScale(scale, "EmbeddingGrad");
  CheckIndex(index, "EmbeddingGrad", "index");
  TORCH_CHECK(grad.device() == index.device(), "EmbeddingGrad: grad and index live on different devices");
  TORCH_CHECK(grad.dim() == index.dim() + 1 && grad.sizes().slice(0, index.dim()) == index.sizes(),
              "EmbeddingGrad: grad must have the shape of index and one more dimension");
  TORCH_CHECK(num_rows >= 0 && num_rows < 0xFFFFFFFFll, "EmbeddingGrad: the table must have fewer than 2^32 - 1 rows");
  TORCH_CHECK(index.numel() < (1ll << 31), "EmbeddingGrad: at most 2^31 - 1 ids a call");
}

torch::Tensor EmbeddingGrad(torch::Tensor grad, torch::Tensor index, int64_t num_rows, double scale, int64_t padding) {
  const int dt = ValueType(grad, "EmbeddingGrad", "grad");
  CheckEmbeddingGrad(grad, index, num_rows, scale);
  c10::cuda::CUDAGuard guard(index.device());
  grad = grad.contiguous();
  index = index.contiguous();
  const int64_t n = index.numel(), D = grad.size(-1);
  auto out = torch::empty({num_rows, D}, grad.options());
  auto ws = NewWorkspace(gsb_embedding_grad_workspace_bytes(n, num_rows, D), index.device());
  CheckStatus(gsb_embedding_grad(grad.data_ptr(), dt, D, index.data_ptr<int64_t>(), n, num_rows, (float)scale, padding,
                                 out.data_ptr(), ws.data_ptr(), (size_t)ws.numel(), ErrorWord(index.device()),
                                 CurrentStream()),
              "embedding_grad");
  return out;
}

std::tuple<torch::Tensor, torch::Tensor> EmbeddingSparseGrad(torch::Tensor grad, torch::Tensor index, int64_t num_rows,
                                                             double scale, int64_t padding) {
  const int dt = ValueType(grad, "EmbeddingSparseGrad", "grad");
  CheckEmbeddingGrad(grad, index, num_rows, scale);
  c10::cuda::CUDAGuard guard(index.device());
  grad = grad.contiguous();
  index = index.contiguous();
  const int64_t n = index.numel(), D = grad.size(-1);
  if (n == 0) return {torch::empty({0}, index.options()), torch::empty({0, D}, grad.options())};
  auto ws = NewWorkspace(gsb_embedding_grad_workspace_bytes(n, num_rows, D), index.device());
  auto ids = torch::empty({n}, index.options());
  auto num = torch::empty({1}, index.options());
  CheckStatus(gsb_embedding_sort(index.data_ptr<int64_t>(), n, num_rows, D, padding, ids.data_ptr<int64_t>(),
                                 num.data_ptr<int64_t>(), ws.data_ptr(), (size_t)ws.numel(), ErrorWord(index.device()),
                                 CurrentStream()),
              "embedding_sort");
  const int64_t U = num.item<int64_t>();
  auto rows = torch::empty({U, D}, grad.options());
  CheckStatus(gsb_embedding_grad_rows(grad.data_ptr(), dt, D, n, num_rows, U, (float)scale, rows.data_ptr(),
                                      ws.data_ptr(), (size_t)ws.numel(), CurrentStream()),
              "embedding_grad_rows");
  return {ids.narrow(0, 0, U).clone(), rows};
}

// ------------------------------------------------------------------ dropout
torch::Tensor Dropout(torch::Tensor data, double p, int64_t seed, int64_t stream, c10::optional<torch::Tensor> step) {
  const int dt = ValueType(data, "Dropout", "data");
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "Dropout: p must lie in [0, 1], got ", p);
  c10::cuda::CUDAGuard guard(data.device());
  const int64_t* step_ptr = nullptr;
  if (step.has_value()) {
    CheckIndex(*step, "Dropout", "step");
    TORCH_CHECK(step->numel() == 1 && step->device() == data.device(),
                "Dropout: step must have one element on data's device");
    step_ptr = step->data_ptr<int64_t>();
  }
  data = data.contiguous();
  auto out = torch::empty(data.sizes(), data.options());
  CheckStatus(gsb_dropout(data.data_ptr(), dt, data.numel(), p, (uint64_t)seed, (uint32_t)stream, step_ptr,
                          out.data_ptr(), CurrentStream()),
              "dropout");
  return out;
}

static std::mutex g_dropout_mutex;
// Not the 7777 that graphs and list sampling start from: with equal seed and stream, element block g of a mask is
// the very words that chose for sampling slot g.
static uint64_t g_dropout_seed = 0x64726F706F757400ull + 7777;
static uint32_t g_dropout_calls = 0;

void SetDropoutSeed(int64_t seed) {
  std::lock_guard<std::mutex> lock(g_dropout_mutex);
  g_dropout_seed = (uint64_t)seed;
  g_dropout_calls = 0;
}

std::tuple<int64_t, int64_t> NextDropoutStream() {
  std::lock_guard<std::mutex> lock(g_dropout_mutex);
  return {(int64_t)g_dropout_seed, (int64_t)g_dropout_calls++};
}

// ------------------------------------------------------------------ vocabulary cross entropy
// rows of a matrix may be strided; anything else is copied
static torch::Tensor Rows(torch::Tensor t) {
  if (t.size(1) > 1 && t.stride(1) != 1) return t.contiguous();
  if (t.size(0) > 1 && t.stride(0) < t.size(1)) return t.contiguous();
  return t;
}
static int64_t RowStep(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

static int CheckLoss(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& target, double scale) {
  const char* op = "LinearCrossEntropy";
  const int dt = ValueType(x, op, "x");
  ValueType(weight, op, "weight");
  CheckIndex(target, op, "target");
  TORCH_CHECK(x.scalar_type() == weight.scalar_type(), op, ": x and weight have different types");
  TORCH_CHECK(x.device() == weight.device() && x.device() == target.device(), op,
              ": x, weight and target live on different devices");
  TORCH_CHECK(x.dim() == 2 && weight.dim() == 2 && x.size(1) == weight.size(1), op,
              ": x must be [N, D] and weight [V, D], got ", x.sizes(), " and ", weight.sizes());
  TORCH_CHECK(target.dim() == 1 && target.size(0) == x.size(0), op, ": target must be [N]");
  TORCH_CHECK(weight.size(0) >= 1 && weight.size(1) >= 1, op, ": weight must have a row and a column");
  TORCH_CHECK(weight.size(1) <= GSB_LOSS_MAX_D, op, ": at most ", GSB_LOSS_MAX_D, " columns");
  TORCH_CHECK(x.size(0) <= (1ll << 30) && weight.size(0) <= (1ll << 30), op, ": at most 2^30 rows");
  CheckScale(scale, op);
  return dt;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> LinearCrossEntropy(torch::Tensor x, torch::Tensor weight,
                                                                           torch::Tensor target, double scale,
                                                                           int64_t ignore, bool want_dx) {
  const int dt = CheckLoss(x, weight, target, scale);
  c10::cuda::CUDAGuard guard(x.device());
  x = Rows(x);
  weight = Rows(weight);
  target = target.contiguous();
  const int64_t N = x.size(0), V = weight.size(0), D = x.size(1);
  auto f32 = x.options().dtype(torch::kFloat32);
  auto loss = torch::empty({N}, f32), lse2 = torch::empty({N}, f32);
  const bool want_pull = want_dx && gsb_linear_ce_has_pull(dt, V, D);
  auto pull = torch::empty(want_pull ? std::vector<int64_t>{N, D} : std::vector<int64_t>{0}, f32);
  auto ws = NewWorkspace(gsb_linear_ce_workspace_bytes(dt, weight.data_ptr(), RowStep(weight), N, V, D, want_pull), x.device());
  CheckStatus(gsb_linear_ce(x.data_ptr(), dt, RowStep(x), N, weight.data_ptr(), RowStep(weight), V, D,
                            target.data_ptr<int64_t>(), ignore, (float)scale, loss.data_ptr<float>(),
                            lse2.data_ptr<float>(), want_pull ? pull.data_ptr<float>() : nullptr, ws.data_ptr(),
                            (size_t)ws.numel(), ErrorWord(x.device()), CurrentStream()),
              "linear_ce");
  return {loss, lse2, pull};
}

std::tuple<torch::Tensor, torch::Tensor> LinearCrossEntropyTotal(torch::Tensor loss, torch::Tensor target,
                                                                 int64_t vocabulary, int64_t ignore, bool mean) {
  CheckIndex(target, "LinearCrossEntropyTotal", "target");
  TORCH_CHECK(loss.is_cuda() && loss.scalar_type() == torch::kFloat32 && loss.is_contiguous() &&
                  loss.sizes() == target.sizes() && loss.device() == target.device(),
              "LinearCrossEntropyTotal: loss must be the contiguous float32 losses of target's rows");
  c10::cuda::CUDAGuard guard(loss.device());
  target = target.contiguous();
  auto total = torch::empty({}, loss.options()), count = torch::empty({}, loss.options());
  auto ws = NewWorkspace(gsb_linear_ce_total_workspace_bytes(loss.numel()), loss.device());
  CheckStatus(gsb_linear_ce_total(loss.data_ptr<float>(), target.data_ptr<int64_t>(), ignore, vocabulary, loss.numel(),
                                  mean, total.data_ptr<float>(), count.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(),
                                  CurrentStream()),
              "linear_ce_total");
  return {total, count};
}

// with the rows' losses, or (undefined) without them
static std::tuple<torch::Tensor, torch::Tensor> GradRows(torch::Tensor x, torch::Tensor weight, torch::Tensor target,
                                                         torch::Tensor rows, torch::Tensor lse2, torch::Tensor pull,
                                                         torch::Tensor upstream, c10::optional<torch::Tensor> count,
                                                         double scale, int64_t ignore, bool want_dx, bool want_dw) {
  const int dt = CheckLoss(x, weight, target, scale);
  const int64_t N = x.size(0), V = weight.size(0), D = x.size(1);
  auto good = [&](const torch::Tensor& t, int64_t n) {
    return t.is_cuda() && t.device() == x.device() && t.scalar_type() == torch::kFloat32 && t.numel() == n;
  };
  const bool per_row = upstream.dim() == 1;
  TORCH_CHECK(good(lse2, N) && lse2.is_contiguous(), "LinearCrossEntropyGrad: lse2 must be float32 [N]");
  TORCH_CHECK(!rows.defined() || (good(rows, N) && rows.is_contiguous()), "LinearCrossEntropyGrad: losses must be float32 [N]");
  const bool have_pull = pull.numel() > 0;
  TORCH_CHECK(!have_pull || (good(pull, N * D) && pull.is_contiguous()), "LinearCrossEntropyGrad: pull must be float32 [N, D]");
  TORCH_CHECK(good(upstream, per_row ? N : 1), "LinearCrossEntropyGrad: upstream must be float32, one value or [N]");
  TORCH_CHECK(!count.has_value() || good(*count, 1), "LinearCrossEntropyGrad: count must be one float32 value");
  c10::cuda::CUDAGuard guard(x.device());
  x = Rows(x);
  weight = Rows(weight);
  target = target.contiguous();
  upstream = upstream.contiguous();
  auto dx = want_dx ? torch::empty({N, D}, x.options()) : torch::empty({0}, x.options());
  auto dw = want_dw ? torch::empty({V, D}, x.options()) : torch::empty({0}, x.options());
  auto ws = NewWorkspace(gsb_linear_ce_grad_workspace_bytes(dt, weight.data_ptr(), RowStep(weight), N, V, D, have_pull, want_dx,
                                                            want_dw),
                         x.device());
  CheckStatus(gsb_linear_ce_grad_rows(x.data_ptr(), dt, RowStep(x), N, weight.data_ptr(), RowStep(weight), V, D,
                                      target.data_ptr<int64_t>(), ignore, (float)scale,
                                      rows.defined() ? rows.data_ptr<float>() : nullptr, lse2.data_ptr<float>(),
                                      have_pull ? pull.data_ptr<float>() : nullptr, upstream.data_ptr<float>(), per_row,
                                      count.has_value() ? count->data_ptr<float>() : nullptr, want_dx ? dx.data_ptr() : nullptr,
                                      want_dw ? dw.data_ptr() : nullptr, ws.data_ptr(), (size_t)ws.numel(), ErrorWord(x.device()),
                                      CurrentStream()),
              "linear_ce_grad");
  return {dx, dw};
}

std::tuple<torch::Tensor, torch::Tensor> LinearCrossEntropyGrad(torch::Tensor x, torch::Tensor weight,
                                                                torch::Tensor target, torch::Tensor lse2,
                                                                torch::Tensor pull, torch::Tensor upstream,
                                                                c10::optional<torch::Tensor> count, double scale,
                                                                int64_t ignore, bool want_dx, bool want_dw) {
  return GradRows(x, weight, target, torch::Tensor(), lse2, pull, upstream, count, scale, ignore, want_dx, want_dw);
}

// ------------------------------------------------------------------ autograd
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

static bool Tracked(const torch::Tensor& t) { return at::GradMode::is_enabled() && t.defined() && t.requires_grad(); }

// The kernels know no tangents and would drop them without a word.
static void RefuseTangent(const torch::Tensor& t, const char* op) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), op, ": forward-mode differentiation is not provided");
}

// The gradient of the lookup is linear in the upstream gradient, and its own gradient is the lookup.
struct EmbeddingGradFn : public torch::autograd::Function<EmbeddingGradFn> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor grad, torch::Tensor index, int64_t rows, double scale,
                               int64_t padding) {
    ctx->save_for_backward({index});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return EmbeddingGrad(grad, index, rows, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    auto up = EmbeddingLookup(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["scale"].toDouble(),
                              ctx->saved_data["padding"].toInt(), /*sparse=*/false);
    return {up, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

static torch::Tensor SparseRows(torch::Tensor grad, torch::Tensor index, int64_t rows, double scale, int64_t padding) {
  torch::Tensor ids, values;
  std::tie(ids, values) = EmbeddingSparseGrad(grad, index, rows, scale, padding);
  return at::_sparse_coo_tensor_unsafe(ids.unsqueeze(0), values, {rows, values.size(1)},
                                       values.options().layout(at::kSparse), /*is_coalesced=*/true);
}

// Under create_graph: a gradient that cannot be differentiated again says so when that is tried, instead of
// counting as a constant.
struct EmbeddingSparseGradFn : public torch::autograd::Function<EmbeddingSparseGradFn> {
  static torch::Tensor forward(AutogradContext*, torch::Tensor grad, torch::Tensor index, int64_t rows, double scale,
                               int64_t padding) {
    return SparseRows(grad, index, rows, scale, padding);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "Embedding: gradients of gradients are not provided for the sparse form");
  }
};

struct EmbeddingFn : public torch::autograd::Function<EmbeddingFn> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor weight, torch::Tensor index, double scale,
                               int64_t padding, bool sparse) {
    auto out = Embedding(weight, index, scale, padding);
    ctx->save_for_backward({index});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["sparse"] = sparse;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto index = ctx->get_saved_variables()[0];
    const int64_t rows = ctx->saved_data["rows"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    torch::Tensor dw;
    if (ctx->saved_data["sparse"].toBool()) {
      dw = Tracked(grads[0]) ? EmbeddingSparseGradFn::apply(grads[0], index, rows, scale, padding)
                             : SparseRows(grads[0], index, rows, scale, padding);
    } else if (Tracked(grads[0])) {
      dw = EmbeddingGradFn::apply(grads[0], index, rows, scale, padding);
    } else {
      dw = EmbeddingGrad(grads[0], index, rows, scale, padding);
    }
    return {dw, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

torch::Tensor EmbeddingLookup(torch::Tensor weight, torch::Tensor index, double scale, int64_t padding, bool sparse) {
  RefuseTangent(weight, "Embedding");
  if (!Tracked(weight)) return Embedding(weight, index, scale, padding);
  return EmbeddingFn::apply(weight, index, scale, padding, sparse);
}

struct DropoutFn : public torch::autograd::Function<DropoutFn> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor data, double p, int64_t seed, int64_t stream,
                               c10::optional<torch::Tensor> step) {
    if (step.has_value()) ctx->save_for_backward({*step});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["stream"] = stream;
    return Dropout(data, p, seed, stream, step);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    c10::optional<torch::Tensor> step;
    if (!saved.empty()) step = saved[0];
    // the same map again, and so is its own gradient
    auto dx = DropoutApply(grads[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                           ctx->saved_data["stream"].toInt(), step);
    return {dx, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

torch::Tensor DropoutApply(torch::Tensor data, double p, c10::optional<int64_t> seed, c10::optional<int64_t> stream,
                           c10::optional<torch::Tensor> step) {
  TORCH_CHECK(seed.has_value() == stream.has_value(), "Dropout: give both seed and stream, or neither");
  RefuseTangent(data, "Dropout");
  int64_t s, t;
  if (seed.has_value()) std::tie(s, t) = std::make_tuple(*seed, *stream);
  else std::tie(s, t) = NextDropoutStream();
  if (!Tracked(data)) return Dropout(data, p, s, t, step);
  return DropoutFn::apply(data, p, s, t, step);
}

// Under create_graph, as above.
struct LinearCrossEntropyGradFn : public torch::autograd::Function<LinearCrossEntropyGradFn> {
  static variable_list forward(AutogradContext*, torch::Tensor x, torch::Tensor weight, torch::Tensor target, torch::Tensor rows,
                               torch::Tensor lse2, torch::Tensor pull, torch::Tensor upstream, c10::optional<torch::Tensor> count, double scale,
                               int64_t ignore, bool want_dx, bool want_dw) {
    torch::Tensor dx, dw;
    std::tie(dx, dw) = GradRows(x, weight, target, rows, lse2, pull, upstream, count, scale, ignore, want_dx, want_dw);
    return {dx, dw};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "LinearCrossEntropy: gradients of gradients are not provided");
  }
};

struct LinearCrossEntropyFn : public torch::autograd::Function<LinearCrossEntropyFn> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor x, torch::Tensor weight, torch::Tensor target,
                               double scale, int64_t ignore, int64_t reduction, bool want_dx) {
    torch::Tensor loss, lse2, pull, count;
    std::tie(loss, lse2, pull) = LinearCrossEntropy(x, weight, target, scale, ignore, want_dx);
    // the backward pass has 1 - p_t from the rows' losses; the ones that go out are the caller's to change
    const auto rows = reduction == 0 ? loss.clone() : loss;
    if (reduction != 0)
      std::tie(loss, count) = LinearCrossEntropyTotal(loss, target, weight.size(0), ignore, reduction == 2);
    if (reduction != 2) count = torch::Tensor();
    ctx->save_for_backward({x, weight, target, lse2, pull, count, rows});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["ignore"] = ignore;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const bool want_dx = ctx->needs_input_grad(0), want_dw = ctx->needs_input_grad(1);
    c10::optional<torch::Tensor> count;
    if (s[5].defined()) count = s[5];
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t ignore = ctx->saved_data["ignore"].toInt();
    torch::Tensor dx, dw;
    if (at::GradMode::is_enabled()) {
      const auto both = LinearCrossEntropyGradFn::apply(s[0], s[1], s[2], s[6], s[3], s[4], grads[0], count, scale, ignore, want_dx, want_dw);
      std::tie(dx, dw) = std::make_tuple(both[0], both[1]);
    } else {
      std::tie(dx, dw) = GradRows(s[0], s[1], s[2], s[6], s[3], s[4], grads[0], count, scale, ignore, want_dx, want_dw);
    }
    return {want_dx ? dx : torch::Tensor(), want_dw ? dw : torch::Tensor(), torch::Tensor(), torch::Tensor(),
            torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

torch::Tensor LinearCrossEntropyLoss(torch::Tensor x, torch::Tensor weight, torch::Tensor target, double scale,
                                     int64_t ignore, int64_t reduction) {
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "LinearCrossEntropy: reduction must be 0, 1 or 2");
  RefuseTangent(x, "LinearCrossEntropy");
  RefuseTangent(weight, "LinearCrossEntropy");
  if (Tracked(x) || Tracked(weight))
    return LinearCrossEntropyFn::apply(x, weight, target, scale, ignore, reduction, Tracked(x));
  auto loss = std::get<0>(LinearCrossEntropy(x, weight, target, scale, ignore, false));
  if (reduction == 0) return loss;
  return std::get<0>(LinearCrossEntropyTotal(loss, target, weight.size(0), ignore, reduction == 2));
}

}  // namespace gsb_host
