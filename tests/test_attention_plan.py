"""Which attention kernels are built, and which of them a call takes, as the
library decides it on the host (no GPU).
"""
import ctypes
import re

import pytest

from pytorch_cluster_amd import _native

WIDTHS = (32, 48, 64, 96, 128)
SIZES = {"f": 4, "DF16_": 2, "DF16b": 2}
PASSES = ("forward", "dq", "dkv")


def plan(kind, nq, nk, hq, hk, size, d):
    """(rows of a workgroup, pieces): pca::AttentionPlan attention_plan(int pass,
    int64_t nq, int64_t nk, int hq, int hk, int size, int d)."""
    function = getattr(ctypes.CDLL(_native.CAPI_PATH),
                       "_ZN3pca14attention_planEilliiii")
    function.restype = ctypes.c_uint64  # two ints
    function.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int64] \
        + 4 * [ctypes.c_int]
    both = function(PASSES.index(kind), nq, nk, hq, hk, size, d)
    return both & 0xffffffff, both >> 32


def test_every_kernel_that_is_built_is_taken():
    text = open(_native.CAPI_PATH, "rb").read()
    built = set(re.findall(
        rb"attention_(forward|dq|dkv)_kernelI(f|DF16_|DF16b)"
        rb"Li(\d+)ELi(\d)ELi(\d)EEEvNS_13AttentionCallE", text))
    built = {(p.decode(), t.decode(), int(w), int(rb), int(wk))
             for p, t, w, rb, wk in built}
    assert built, "no kernels found"
    taken = set()
    kernel = {16: (1, 4), 64: (1, 1), 128: (2, 1)}
    for kind in PASSES:
        for name, size in SIZES.items():
            for w in WIDTHS:
                for n in (20, 5000, 1000000):
                    rows, _ = plan(kind, n, n, 8, 8, size, w)
                    taken.add((kind, name, w) + kernel[rows])
    assert built == taken
