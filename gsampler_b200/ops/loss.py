"""Softmax cross entropy over a vocabulary of nodes (or classes) that never holds the logits: the last
step of training on walks (the next node out of all of them) and of node classification."""
import torch

__all__ = ["linear_cross_entropy"]


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, scale, ignore_index, reduction):
        loss, lse2, pull = torch.ops.gs_ops._CAPI_LinearCrossEntropy(x, weight, target, scale, ignore_index,
                                                                     ctx.needs_input_grad[0])
        count = None
        if reduction != "none":
            loss, count = torch.ops.gs_ops._CAPI_LinearCrossEntropyTotal(loss, target, weight.shape[0], ignore_index,
                                                                         reduction == "mean")
        ctx.save_for_backward(x, weight, target, lse2, pull, count if reduction == "mean" else None)
        ctx.scale, ctx.ignore_index = scale, ignore_index
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, target, lse2, pull, count = ctx.saved_tensors
        want_dx, want_dw = ctx.needs_input_grad[:2]
        dx, dw = torch.ops.gs_ops._CAPI_LinearCrossEntropyGrad(x, weight, target, lse2, pull, grad, count, ctx.scale,
                                                               ctx.ignore_index, want_dx, want_dw)
        return dx if want_dx else None, dw if want_dw else None, None, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, scale: float = 1.0,
                         ignore_index: int = -1, reduction: str = "mean") -> torch.Tensor:
    """``-log softmax(scale * x @ weight.T)[target]`` for representations ``x`` [..., D], a vocabulary
    ``weight`` [V, D] of the same type (fp32, fp16 or bf16) and int64 ``target`` [...].

    The logits are made piece by piece and never stored, in either pass.  The loss is fp32:
    ``reduction`` "mean" (over the rows that count), "sum", or "none" (every row's, which is also how a
    single row is scored when serving).  A row whose target is ``ignore_index`` does not count: its
    loss and gradients are zero, whatever ``x`` holds there; "mean" over no rows is zero.  A target
    outside the vocabulary does not count either and is reported by ``check_async_errors()``.
    Nothing here synchronises."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("linear_cross_entropy: reduction must be mean, sum or none, got %r" % (reduction,))
    if x.dim() < 1 or x.shape[:-1] != target.shape:
        raise ValueError("linear_cross_entropy: target must have the shape of x without its last dimension")
    loss = _LinearCrossEntropy.apply(x.reshape(-1, x.shape[-1]), weight, target.reshape(-1), float(scale),
                                     int(ignore_index), reduction)
    return loss.view(target.shape) if reduction == "none" else loss
