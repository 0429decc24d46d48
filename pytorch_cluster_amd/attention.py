"""``attention``: softmax attention between the rows of the same example.

The reference has no counterpart; the operator stands next to ``knn`` and
``radius``, which compare the same pairs of rows, and takes examples as they
do: sorted batch vectors, no padding.  Stays ``torch.jit.script``-able.  GPU
tensors only.
"""
from typing import Optional

import torch


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    batch_q: Optional[torch.Tensor] = None,
    batch_k: Optional[torch.Tensor] = None,
    pos_q: Optional[torch.Tensor] = None,
    pos_k: Optional[torch.Tensor] = None,
    slope: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    cap: float = 0.0
) -> torch.Tensor:
    r"""Each row of ``q`` looks at all rows of ``k`` of the same example:
    ``out[i, h] = sum_j softmax_j(s_ij) v[j, h']`` with ``s_ij = u(scale *
    q[i, h] . k[j, h']) - slope[h] * |pos_q[i] - pos_k[j]|``.

    Args:
        q: ``[M, H, C]`` queries, float32, float16 or bfloat16, ``C <= 128``.
        k: ``[N, H', C]`` keys; ``H`` is a multiple of ``H'``, and ``H / H'``
            neighbouring heads of ``q`` share a head of ``k`` and ``v``.
        v: ``[N, H', C]`` values.  Strided views are read in place as long as
            their last dimension is dense.
        batch_q: sorted ``[M]`` vector assigning each query to an example;
            together with ``batch_k``.  An unsorted vector is not detected.
        batch_k: the same for ``k`` and ``v``.  A query whose example has no
            row in ``k`` returns zeros, and so does one whose scores are all
            ``-inf``.
        pos_q: ``[M, 1 to 3]`` float32 positions of the queries, for the bias by
            distance; no gradient.
        pos_k: the same for ``k``.
        slope: ``[H]`` float32, what a unit of (Euclidean) distance takes off
            the score; no gradient.
        scale: factor of the products (default ``C ** -0.5``).
        cap: if positive, products are bounded before the bias is added:
            ``u(t) = cap * tanh(t / cap)``; any size (above ``2 ** 127`` that
            counts).

    Returns ``[M, H, C]`` of ``q``'s type.  ``q``, ``k`` and ``v`` get gradients
    (once: second and forward-mode derivatives raise).

    Scores, softmax statistics and sums are held in 32 bits.  With 16-bit rows
    the weights, and in the backward pass the scores' gradients, are rounded
    once to that type for the matrix cores; float32 rows round nothing below
    32 bits.  The same call gives the same bits.  May be captured into a graph;
    as with any operator of torch, a backward pass is captured while no eager
    graph of the same leaves is alive.
    """
    return torch.ops.pytorch_cluster_amd.attention(
        q, k, v, batch_q, batch_k, pos_q, pos_k, slope, scale, cap)
