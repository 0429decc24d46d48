"""``norm_rotate``: norm of queries and keys per head and rotation by the rows'
positions, in one pass: what makes the ``q`` and ``k`` of ``attention``.

No counterpart in the reference.  Stays ``torch.jit.script``-able.  GPU tensors
only.
"""
from typing import Optional, Tuple

import torch


def norm_rotate(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    pos: torch.Tensor,
    freq: torch.Tensor,
    weight_q: Optional[torch.Tensor] = None,
    weight_k: Optional[torch.Tensor] = None,
    eps: float = 1e-6
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    r"""``y = weight * x / sqrt(mean(x ** 2) + eps)`` over the channels of each
    head, then pairs ``(c, c + R)`` of ``y`` turned by the angle ``sum_p pos[:,
    p] * freq[p, c]``; channels from ``2 R`` on are not turned.

    Args:
        q: ``[N, H, C]``, float32, float16 or bfloat16, ``C <= 256``.
        k: ``[N, H', C]`` of the same type, or ``None``.
        pos: ``[N, P]`` float32 positions, 1 to 3 axes; no gradient.
        freq: ``[P, R]`` float32, ``2 R <= C``, radians per unit of position;
            no gradient.  Angles are formed in 64 bits.
        weight_q: ``[C]`` gain of ``q`` (default ones), of ``q``'s type or
            float32.
        weight_k: the same for ``k``.
        eps: added to the mean square, which is formed in 32 bits: components
            beyond ``1e18``, or without ``eps`` all below ``1e-18``, leave its
            range.

    Returns ``q`` and ``k`` (or ``None``) normed and turned.  ``q``, ``k`` and
    the weights get gradients (once: second and forward-mode derivatives
    raise).
    """
    outs = torch.ops.pytorch_cluster_amd.norm_rotate(q, k, pos, freq, weight_q,
                                                     weight_k, eps)
    turned_k: Optional[torch.Tensor] = None
    if len(outs) > 1:
        turned_k = outs[1]
    return outs[0], turned_k
