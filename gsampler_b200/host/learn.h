// Operators on learned node values behind torch.ops.gs_ops.*: embedding lookup, dropout and the
// softmax cross entropy over a vocabulary, each with its gradient.  They have no counterpart in
// the reference, whose examples hand these steps to torch.
#pragma once
#include <torch/script.h>

#include <tuple>

namespace gsb_host {

torch::Tensor Embedding(torch::Tensor weight, torch::Tensor index, double scale, int64_t padding);
torch::Tensor EmbeddingGrad(torch::Tensor grad, torch::Tensor index, int64_t num_rows, double scale, int64_t padding);
// (ids, rows): the touched rows, ids ascending; one read-back (their number)
std::tuple<torch::Tensor, torch::Tensor> EmbeddingSparseGrad(torch::Tensor grad, torch::Tensor index, int64_t num_rows,
                                                             double scale, int64_t padding);
// `step` (optional one-element int64 tensor on the GPU) is added to `stream` when the kernel runs
torch::Tensor Dropout(torch::Tensor data, double p, int64_t seed, int64_t stream, c10::optional<torch::Tensor> step);
// default random state of dropout: a seed (its own, not the samplers') and a per-process call counter
void SetDropoutSeed(int64_t seed);
std::tuple<int64_t, int64_t> NextDropoutStream();

// softmax cross entropy over a vocabulary: (loss of every row, log-sum-exp of every row in base 2, and
// -- empty unless asked for and available -- what the gradient of x is made from)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> LinearCrossEntropy(torch::Tensor x, torch::Tensor weight,
                                                                           torch::Tensor target, double scale,
                                                                           int64_t ignore, bool want_dx);
// (sum or mean of the rows' losses, number of rows that count)
std::tuple<torch::Tensor, torch::Tensor> LinearCrossEntropyTotal(torch::Tensor loss, torch::Tensor target,
                                                                 int64_t vocabulary, int64_t ignore, bool mean);
// (dx, dw); one that is not asked for comes back empty
std::tuple<torch::Tensor, torch::Tensor> LinearCrossEntropyGrad(torch::Tensor x, torch::Tensor weight,
                                                                torch::Tensor target, torch::Tensor lse2,
                                                                torch::Tensor pull, torch::Tensor upstream,
                                                                c10::optional<torch::Tensor> count, double scale,
                                                                int64_t ignore, bool want_dx, bool want_dw);

// The same with their gradients, for autograd (reverse mode; gradients of gradients for the lookup with a dense
// gradient and for dropout, an error for the others).
torch::Tensor EmbeddingLookup(torch::Tensor weight, torch::Tensor index, double scale, int64_t padding, bool sparse);
// dropout without seed and stream takes them from the default state when it runs
torch::Tensor DropoutApply(torch::Tensor data, double p, c10::optional<int64_t> seed, c10::optional<int64_t> stream,
                           c10::optional<torch::Tensor> step);
// reduction: 0 none, 1 sum, 2 mean
torch::Tensor LinearCrossEntropyLoss(torch::Tensor x, torch::Tensor weight, torch::Tensor target, double scale,
                                     int64_t ignore, int64_t reduction);

}  // namespace gsb_host
