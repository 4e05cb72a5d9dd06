"""Dropout from the library's counter-based random streams: the mask is a function of (seed,
stream, element), so it is never stored and the backward pass draws it again."""
import torch

__all__ = ["dropout"]


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, data, p, seed, stream, step):
        ctx.p, ctx.seed, ctx.stream = p, seed, stream
        ctx.save_for_backward(*([] if step is None else [step]))
        return torch.ops.gs_ops._CAPI_Dropout(data, p, seed, stream, step)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        step = ctx.saved_tensors[0] if ctx.saved_tensors else None
        return torch.ops.gs_ops._CAPI_Dropout(grad, ctx.p, ctx.seed, ctx.stream, step), None, None, None, None


def dropout(data: torch.Tensor, p: float = 0.5, training: bool = True, seed: int = None, stream: int = None,
            step: torch.Tensor = None) -> torch.Tensor:
    """Zeroes each element of ``data`` (fp32, fp16 or bf16) with probability ``p`` and multiplies the
    others by the inverse of the kept share.  ``p`` is taken to the nearest 1/65536, and the factor
    belongs to that value.  ``training=False`` or ``p == 0`` returns ``data`` itself.

    The mask depends on ``seed``, ``stream`` and the element's position in row-major order only.
    Left out, they come from the process's dropout state: the seed of
    ``torch.ops.gs_ops._CAPI_SetDropoutSeed`` (default 7777) and a counter that advances with every
    call.  Give both to repeat a mask.  A recorded CUDA graph replays the recorded streams; ``step``, a
    one-element int64 tensor on the GPU that is added to ``stream`` when the kernel runs, gives
    every replay a mask of its own (advance it after the backward pass, which reads it again)."""
    if (seed is None) != (stream is None):
        raise ValueError("dropout: give both seed and stream, or neither")
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout: p must lie in [0, 1], got %s" % (p,))
    if not training or p == 0.0:
        return data
    if seed is None:
        seed, stream = torch.ops.gs_ops._CAPI_NextDropoutStream()
    return _Dropout.apply(data, float(p), int(seed), int(stream), step)
