from .spmm import gspmm
from .sddmm import gsddmm
from .fused import e_square_sum, e_div_u_sum
from .embedding import embedding
from .dropout import dropout
from .loss import linear_cross_entropy

__all__ = ["gspmm", "gsddmm", "e_square_sum", "e_div_u_sum", "embedding", "dropout", "linear_cross_entropy"]
