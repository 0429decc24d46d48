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


def many_rows():
    """Sizes of 64 examples, of none to 400 rows, in which rows of several examples
    share a tile: at 8 key heads enough for 128 rows a workgroup."""
    sizes = [(37 * i * i + 11 * i) % 401 for i in range(64)]
    sizes[5], sizes[6], sizes[7] = 1, 0, 2
    return sizes


# Heads of which some pass has kernels of 128 rows, and what is cut into pieces: type
# (size), width, pass.
WIDE_TILES = [(2, 33, "dkv"), (2, 48, "dkv"), (2, 63, "dkv"), (2, 64, "dkv"),
              (2, 65, "forward"), (2, 96, "forward"), (2, 100, "forward"),
              (2, 127, "forward"), (2, 128, "forward")] + [
    (4, d, p) for d in (33, 48, 57, 64) for p in PASSES]


@pytest.mark.parametrize("size,d,kind", WIDE_TILES)
@pytest.mark.parametrize("heads", [8, 16])
def test_many_rows_take_tiles_of_128(size, d, kind, heads):
    n = sum(many_rows())
    assert plan(kind, n, n, heads, 8, size, d) == (128, 1)


# Rows and heads whose looped side is cut into pieces of tiles of 16 and of 64 rows.
CUT = [(1100, 2), (100, 1)]


@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("d", [5, 31, 65, 127])
@pytest.mark.parametrize("kind", PASSES)
@pytest.mark.parametrize("owned,heads", CUT)
def test_few_rows_are_cut_into_pieces(size, d, kind, owned, heads):
    sides = (owned, 2300) if kind != "dkv" else (2300, owned)
    rows, pieces = plan(kind, *sides, heads, heads, size, d)
    assert rows == (16 if owned <= 256 else 64) and pieces > 1
