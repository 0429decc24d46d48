"""attention, norm_rotate and lookup without a GPU: what they refuse, the C ABI's
own checks, exported symbols, TorchScript.
"""
import ctypes
import os
import re

import pytest
import torch

import pytorch_cluster_amd as pca
from pytorch_cluster_amd import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_symbols_are_exported():
    header = open(os.path.join(ROOT, "include", "pca_features.h")).read()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    declared = set(re.findall(r"\b(pca_[a-z0-9_]+)\s*\(", header))
    assert declared == set(_native.FEATURES_C_ABI), "ctypes table out of date"
    lib = ctypes.CDLL(_native.CAPI_PATH)
    for name in sorted(declared):
        assert hasattr(lib, name), "missing export: " + name


def test_scriptable():
    for fn in (pca.attention, pca.norm_rotate, pca.lookup):
        torch.jit.script(fn)


def qkv(rows=6, heads=4, d=8, dtype=torch.float32):
    return tuple(torch.zeros(rows, heads, d, dtype=dtype) for _ in range(3))


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(6, 8)), "rows, heads, channels"),
    (dict(q=torch.zeros(6, 4, 8, dtype=torch.float64)), "float32, float16"),
    (dict(k=torch.zeros(6, 4, 8, dtype=torch.float16)), "one type"),
    (dict(v=torch.zeros(5, 4, 8)), "one shape"),
    (dict(q=torch.zeros(6, 4, 9)), "channels, 9 and 8"),
    (dict(q=torch.zeros(6, 6, 8)), "multiple"),
    (dict(q=torch.zeros(6, 0, 8)), "multiple"),
    (dict(batch_q=torch.zeros(6, dtype=torch.long)), "go together"),
    (dict(batch_q=torch.zeros(6, dtype=torch.long),
          batch_k=torch.zeros(5, dtype=torch.long)), "one entry for each row"),
    (dict(batch_q=torch.zeros(6), batch_k=torch.zeros(6)), "integers"),
    (dict(slope=torch.zeros(4)), "go together"),
    (dict(slope=torch.zeros(4), pos_q=torch.zeros(6, 3),
          pos_k=torch.zeros(6, 2)), "differ in their axes"),
    (dict(slope=torch.zeros(4), pos_q=torch.zeros(6, 4),
          pos_k=torch.zeros(6, 4)), "1 to 3 axes"),
    (dict(slope=torch.zeros(4), pos_q=torch.zeros(5, 3),
          pos_k=torch.zeros(6, 3)), "5 rows for 6"),
    (dict(slope=torch.zeros(4), pos_q=torch.zeros(6, 3).half(),
          pos_k=torch.zeros(6, 3)), "float32"),
    (dict(slope=torch.zeros(3), pos_q=torch.zeros(6, 3),
          pos_k=torch.zeros(6, 3)), "one for each head"),
    (dict(slope=torch.zeros(4, requires_grad=True), pos_q=torch.zeros(6, 3),
          pos_k=torch.zeros(6, 3)), "slope gets no gradient"),
    (dict(slope=torch.zeros(4), pos_q=torch.zeros(6, 3, requires_grad=True),
          pos_k=torch.zeros(6, 3)), "pos_q gets no gradient"),
    (dict(cap=-1.0), "cap"),
    (dict(cap=float("inf")), "cap"),
    (dict(scale=float("nan")), "scale"),
    (dict(), "must be CUDA tensor"),
])
def test_attention_refuses(change, text):
    q, k, v = qkv()
    args = dict(dict(q=q, k=k, v=v), **change)
    with pytest.raises(RuntimeError, match=text):
        pca.attention(**args)


def test_attention_refuses_wide_heads():
    with pytest.raises(RuntimeError, match="1 to 128 channels"):
        pca.attention(*qkv(d=129))


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(6, 8)), "rows, heads, channels"),
    (dict(q=torch.zeros(6, 4, 8, dtype=torch.float64)), "float32, float16"),
    (dict(q=torch.zeros(6, 4, 257)), "1 to 256 channels"),
    (dict(k=torch.zeros(5, 4, 8)), "rows and channels"),
    (dict(k=torch.zeros(6, 4, 8).half()), "of q's type"),
    (dict(pos=torch.zeros(6, 4)), "1 to 3 axes"),
    (dict(pos=torch.zeros(6, 3, dtype=torch.float64)), "float32"),
    (dict(pos=torch.zeros(6, 3, requires_grad=True)), "no gradient"),
    (dict(freq=torch.zeros(2, 4)), "axes of pos, pairs"),
    (dict(freq=torch.zeros(3, 5)), "do not fit"),
    (dict(freq=torch.zeros(3, 4, requires_grad=True)), "no gradient"),
    (dict(weight_k=torch.ones(8)), "weight_k without k"),
    (dict(weight_q=torch.ones(7)), "channels"),
    (dict(weight_q=torch.ones(8).half()), "q's type or"),
    (dict(eps=-1.0), "eps"),
    (dict(), "must be CUDA tensor"),
])
def test_norm_rotate_refuses(change, text):
    args = dict(dict(q=torch.zeros(6, 4, 8), k=None, pos=torch.zeros(6, 3),
                     freq=torch.zeros(3, 4)), **change)
    with pytest.raises(RuntimeError, match=text):
        pca.norm_rotate(**args)


@pytest.mark.parametrize("change,text", [
    (dict(weight=torch.zeros(6)), "rows, channels"),
    (dict(weight=torch.zeros(6, 4, dtype=torch.float64)), "float32, float16"),
    (dict(index=torch.zeros(3)), "int64 or int32"),
    (dict(index=torch.zeros(3, dtype=torch.int16)), "int64 or int32"),
    (dict(scale=float("inf")), "scale"),
    (dict(), "must be CUDA tensor"),
])
def test_lookup_refuses(change, text):
    args = dict(dict(weight=torch.zeros(6, 4),
                     index=torch.zeros(3, dtype=torch.long)), **change)
    with pytest.raises(RuntimeError, match=text):
        pca.lookup(**args)


def test_c_abi_checks_before_any_launch():
    lib = _native.capi
    at = 1 << 20  # (an address that is never used)
    args = _native.AttentionArgs(q=at, k=at, v=at, nq=10, nk=10, hq=4, hk=2,
                                 d=64, dtype=0, scale=1.0, cap=0.0)

    def forward(ws=at, size=1 << 30, out=at, **change):
        a = _native.AttentionArgs.from_buffer_copy(args)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.pca_attention_forward(ctypes.byref(a), out, None, None, ws,
                                         size, None)
    assert lib.pca_attention_forward(None, at, None, None, at, 1 << 20, None) == -1
    assert forward(dtype=1) == -5
    assert forward(d=129) == -5
    assert b"up to 128" in lib.pca_last_error()
    assert forward(d=0) == -1
    assert forward(hq=3) == -1
    assert forward(hk=0) == -1
    assert forward(nq=-1) == -1
    assert forward(nq=2 ** 31 - 2) == -1  # (times two heads of a group)
    assert forward(k=None) == -1
    assert forward(slope=at, axes=2) == -1
    assert forward(slope=at, axes=4, pos_q=at, pos_k=at) == -1
    assert forward(cap=-1.0) == -1
    assert forward(scale=float("nan")) == -1
    assert forward(out=at + 8) == -1
    assert forward(spans_q=at + 4) == -1
    assert forward(size=16) == -3
    assert forward(ws=at + 8) == -3
    assert forward(ws=None) == -3
    assert lib.pca_attention_workspace_bytes(10, 10, 4, 3, 64, 0) == 0
    assert lib.pca_attention_workspace_bytes(10, 10, 4, 2, 64, 1) > 0

    def backward(dq=at, lse=at, **change):
        a = _native.AttentionArgs.from_buffer_copy(args)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.pca_attention_backward(
            ctypes.byref(a), at, None, lse, at, 256, 64, dq, at, at, at,
            1 << 30, None)
    assert backward(lse=None) == -1
    assert backward(dq=None) == -1
    assert backward(dq=at + 2) == -1
    assert backward(spans_q=at) == -1
    assert lib.pca_spans(None, 5, at, 5, at, None) == -1
    assert lib.pca_spans(at, 5, at, 5, at + 4, None) == -1

    rows = _native.NormRotateArgs(q=at, rows=10, hq=2, hk=0, d=16, axes=2,
                                  rotated=8, pos=at, freq=at, dtype=3,
                                  weight_dtype=0, eps=1e-6)

    def rotate(out=at, **change):
        a = _native.NormRotateArgs.from_buffer_copy(rows)
        for name, value in change.items():
            setattr(a, name, value)
        return lib.pca_norm_rotate_forward(ctypes.byref(a), out, None, None)
    assert rotate(dtype=1) == -5
    assert rotate(weight_dtype=1) == -5
    assert rotate(d=257) == -1
    assert rotate(rotated=9) == -1
    assert rotate(axes=0) == -1
    assert rotate(hk=1) == -1
    assert rotate(pos=None) == -1
    assert rotate(eps=-1.0) == -1
    assert rotate(out=None) == -1
    assert rotate(out=at + 4) == -1
    assert lib.pca_norm_rotate_workspace_bytes(10, 300) == 0
    assert lib.pca_norm_rotate_backward(
        ctypes.byref(rows), at, 32, 16, None, 0, 0, at, None, None, None, at,
        16, None) == -3

    def lookup(table=at, size=8, rows=10, entries=5, width=4, dtype=0, out=at):
        return lib.pca_lookup(table, at, size, rows, entries, width, 1.0, dtype,
                              out, None)
    assert lookup(dtype=1) == -5
    assert lookup(size=2) == -1
    assert lookup(rows=-1) == -1
    assert lookup(entries=2 ** 31) == -1
    assert lookup(width=(1 << 20) + 1) == -1
    assert lookup(table=None) == -1
    assert lookup(table=at + 4) == -1
    assert lookup(out=at + 4) == -1
    assert lib.pca_lookup_grad(at, at, 8, 10, 5, 4, 1.0, 0, at, at, 16,
                               None) == -3
