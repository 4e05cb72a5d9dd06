"""Embedding lookup with scaling, and its gradient by sorted ids.

``gather_rows`` fetches features that are given; this is the fetch of values that are learned
(DeepWalk / node2vec tables, graphs without input features): ids come from ``all_nodes()`` or a
walk, -1 marks "no node" as everywhere in this library."""
import torch

__all__ = ["embedding"]


def embedding(weight: torch.Tensor, index: torch.Tensor, scale: float = 1.0, padding_idx: int = -1,
              sparse: bool = False) -> torch.Tensor:
    """``scale * weight[index]`` for a table ``weight`` [rows, D] (fp32, fp16 or bf16) and int64 ids
    of any shape; the result has ``index.shape + (D,)``.

    An id equal to ``padding_idx`` gives a row of zeros and has no gradient.  Any other id outside
    the table does the same and is reported by ``check_async_errors()``; nothing here synchronises.

    The gradient sums the rows of equal ids in 32 bits, in an order that their positions fix (the same
    inputs give the same bits on the same kind of GPU), and rounds once.  ``sparse=True`` returns it as a coalesced sparse
    tensor over the touched rows, which costs one read-back of their number (so it cannot be
    recorded into a CUDA graph); the dense form writes the whole table.  The dense gradient can be
    differentiated again; the sparse one, and forward-mode differentiation, raise."""
    return torch.ops.gs_ops._CAPI_EmbeddingLookup(weight, index, float(scale), int(padding_idx), bool(sparse))
