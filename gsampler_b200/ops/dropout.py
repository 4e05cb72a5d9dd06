"""Dropout from the library's counter-based random streams: the mask is a function of (seed,
stream, element), so it is never stored and the backward pass draws it again."""
import torch

__all__ = ["dropout"]


def dropout(data: torch.Tensor, p: float = 0.5, training: bool = True, seed: int = None, stream: int = None,
            step: torch.Tensor = None) -> torch.Tensor:
    """Zeroes each element of ``data`` (fp32, fp16 or bf16) with probability ``p`` and multiplies the
    others by the inverse of the kept share.  ``p`` is taken to the nearest 1/65536, and the factor
    belongs to that value.  ``training=False`` or ``p == 0`` returns ``data`` itself.

    The mask depends on ``seed``, ``stream`` and the element's position in row-major order only.
    Left out, they come from the process's dropout state: the seed of
    ``torch.ops.gs_ops._CAPI_SetDropoutSeed`` (by default one that no sampler starts from) and a counter
    that advances with every call.  Give both to repeat a mask, also where a forward pass is
    computed twice (activation checkpointing).  A seed that a graph or list sampling uses
    too makes masks of the words that chose there, wherever the stream numbers meet: keep them apart.
    ``stream`` counts modulo 2^32.  A recorded CUDA graph replays the recorded streams; ``step``, a
    one-element int64 tensor on the GPU that is added to ``stream`` when the kernel runs, gives
    every replay a mask of its own (advance it after the backward pass, which reads it again).
    Gradients can be differentiated again; forward-mode differentiation raises."""
    if (seed is None) != (stream is None):
        raise ValueError("dropout: give both seed and stream, or neither")
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout: p must lie in [0, 1], got %s" % (p,))
    if not training or p == 0.0:
        return data
    return torch.ops.gs_ops._CAPI_DropoutApply(data, float(p), seed, stream, step)
