"""What attention, norm_rotate and lookup refuse beyond shapes and types (no GPU):
forward-mode derivatives, numbers at the ends of their types in the C ABI.
"""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

import pytorch_cluster_amd as pca
from pytorch_cluster_amd import _native

AT = 1 << 20  # (an address that is never used)


def arguments(op):
    rows = torch.zeros(6, 4, 8)
    if op == "attention":
        return dict(q=rows, k=rows.clone(), v=rows.clone(),
                    pos_q=torch.zeros(6, 3), pos_k=torch.zeros(6, 3),
                    slope=torch.zeros(4))
    if op == "norm_rotate":
        return dict(q=rows, k=rows.clone(), pos=torch.zeros(6, 3),
                    freq=torch.zeros(3, 4), weight_q=torch.ones(8),
                    weight_k=torch.ones(8))
    return dict(weight=torch.zeros(6, 4), index=torch.zeros(3, dtype=torch.long))


@pytest.mark.parametrize("op,name", [
    (op, n) for op in ("attention", "norm_rotate", "lookup")
    for n, t in arguments(op).items() if t.is_floating_point()])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(op, name, grad):
    args = arguments(op)
    differentiable = name in ("q", "k", "v", "weight_q", "weight_k", "weight")
    with fwd.dual_level():
        primal = args[name].clone().requires_grad_(grad and differentiable)
        args[name] = fwd.make_dual(primal, torch.ones_like(primal))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            getattr(pca, op)(**args)
        with torch.no_grad():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                getattr(pca, op)(**args)
    # (without a tangent: as far as the device)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="must be CUDA tensor"):
            getattr(pca, op)(**arguments(op))


@pytest.mark.parametrize("rotated", [9, 2 ** 30, 2 ** 30 + 5, 2 ** 31 - 1, -1,
                                     -2 ** 30, -2 ** 31])
def test_pairs_that_do_not_fit_a_head(rotated):
    # (twice 2^30 does not fit 32 bits)
    args = _native.NormRotateArgs(q=AT, rows=10, hq=2, hk=0, d=16, axes=2,
                                  rotated=rotated, pos=AT, freq=AT, dtype=3,
                                  weight_dtype=0, eps=1e-6)
    lib = _native.capi
    assert lib.pca_norm_rotate_forward(ctypes.byref(args), AT, None, None) == -1
    size = lib.pca_norm_rotate_workspace_bytes(10, 16)
    assert lib.pca_norm_rotate_backward(
        ctypes.byref(args), AT, 32, 16, None, 0, 0, AT, None, None, None, AT,
        size, None) == -1


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_factors_of_rows_that_are_no_numbers(scale):
    # (times a component of zero: NaN)
    lib = _native.capi
    assert lib.pca_lookup(AT, AT, 8, 10, 5, 4, scale, 0, AT, None) == -1
    assert b"finite" in lib.pca_last_error()
    size = lib.pca_lookup_grad_workspace_bytes(10, 5, 4)
    assert lib.pca_lookup_grad(AT, AT, 8, 10, 5, 4, scale, 0, AT, AT, size,
                               None) == -1


@pytest.mark.parametrize("heads", [1, 2, 7])
@pytest.mark.parametrize("side", ["nq", "nk"])
def test_rows_that_one_launch_cannot_take(heads, side):
    # 64 rows of a key head a workgroup of 256, 2^32 threads in a launch
    most = (2 ** 24 - 1) // heads * 64

    def sizes(n):
        return (n, 5) if side == "nq" else (5, n)

    def workspace(n, backward):
        return _native.capi.pca_attention_workspace_bytes(
            *sizes(n), heads, heads, 1, backward)
    for backward in (0, 1):
        assert workspace(most, backward) > 0
        assert workspace(most + 1, backward) == 0
    nq, nk = sizes(most + 1)
    args = _native.AttentionArgs(q=AT, k=AT, v=AT, nq=nq, nk=nk, hq=heads,
                                 hk=heads, d=1, dtype=0, scale=1.0, cap=0.0)
    assert _native.capi.pca_attention_forward(
        ctypes.byref(args), AT, None, None, AT, 1 << 40, None) == -1
    assert b"out of range" in _native.capi.pca_last_error()
