"""Softmax cross entropy over a vocabulary of nodes (or classes) that never holds the logits: the last
step of training on walks (the next node out of all of them) and of node classification."""
import torch

__all__ = ["linear_cross_entropy"]


_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, scale: float = 1.0,
                         ignore_index: int = -1, reduction: str = "mean") -> torch.Tensor:
    """``-log softmax(scale * x @ weight.T)[target]`` for representations ``x`` [..., D], a vocabulary
    ``weight`` [V, D] of the same type (fp32, fp16 or bf16) and int64 ``target`` [...].

    The logits are made piece by piece and never stored, in either pass.  The loss is fp32:
    ``reduction`` "mean" (over the rows that count), "sum", or "none" (every row's, which is also how a
    single row is scored when serving).  A row whose target is ``ignore_index`` does not count: its
    loss and gradients are zero, whatever ``x`` holds there; "mean" over no rows is zero.  A target
    outside the vocabulary does not count either and is reported by ``check_async_errors()``.
    Nothing here synchronises.  Gradients of gradients and forward-mode differentiation raise."""
    how = _REDUCTIONS.get(reduction)
    if how is None:
        raise ValueError("linear_cross_entropy: reduction must be mean, sum or none, got %r" % (reduction,))
    shape = target.shape
    if x.dim() < 1 or x.shape[:-1] != shape:
        raise ValueError("linear_cross_entropy: target must have the shape of x without its last dimension")
    if x.dim() != 2:
        x, target = x.reshape(-1, x.shape[-1]), target.reshape(-1)
    loss = torch.ops.gs_ops._CAPI_LinearCrossEntropyLoss(x, weight, target, float(scale), int(ignore_index), how)
    return loss.view(shape) if how == 0 else loss
