"""``lookup``: rows by the row numbers that ``knn``, ``radius``, ``nearest`` and
``fps`` return (features of neighbours, entries of a code book, sampled rows),
and the gradient of the table.

No counterpart in the reference.  Stays ``torch.jit.script``-able.  GPU tensors
only.
"""
import torch


def lookup(weight: torch.Tensor, index: torch.Tensor,
           scale: float = 1.0) -> torch.Tensor:
    r"""``out[e] = scale * weight[index[e]]``.

    Args:
        weight: ``[N, C]`` table, float32, float16 or bfloat16.
        index: int64 or int32 row numbers, of any shape.  An entry outside ``0
            .. N - 1`` (``-1`` for a place without a row) reads nothing: its
            output row is zeros and it adds to no gradient.
        scale: factor of the rows.

    Returns ``[*index.shape, C]``.  ``weight`` gets a gradient (once: second
    and forward-mode derivatives raise), summed in 32 bits from the entries in
    the order of their rows: the same call gives the same bits.
    """
    return torch.ops.pytorch_cluster_amd.lookup(weight, index, scale)
