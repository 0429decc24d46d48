"""attention in its kernels of 128 rows and with sides cut into pieces, at widths that
no vector divides, rows that start anywhere, examples that share tiles; and the
backward pass with and without what rounding took off the output.
"""
import ctypes

import pytest
import torch

from pytorch_cluster_amd import _native
from attention_bounds import attention_bounds
from features_common import check
from test_attention_plan import CUT, PASSES, many_rows, plan
from test_gpu_attention import DEV, TYPES, call, inputs

pytestmark = pytest.mark.gpu


def compare(x, **more):
    got = call(x, **more)
    val, err = attention_bounds(**dict(x, **more))
    check(got, val, err)
    return got


def shifted(t):
    """The same values in rows that do not start on 16 bytes."""
    room = torch.empty(t.size(0), t.size(1), t.size(2) + 3, dtype=t.dtype,
                       device=DEV)
    return room[..., 1:-2].copy_(t)


def taken(x):
    d, hq, hk = x["q"].size(2), x["q"].size(1), x["k"].size(1)
    return [plan(p, x["q"].size(0), x["k"].size(0), hq, hk,
                 x["q"].element_size(), d) for p in PASSES]


# ---- 128 rows a workgroup -------------------------------------------------------

def ragged(seed, dtype, d, axes=0, heads=8):
    """As many rows on both sides, of other examples' sizes."""
    sizes = many_rows()
    return inputs(seed, sum(sizes), sum(sizes), heads, 8, d, TYPES[dtype],
                  axes=axes, sizes_q=sizes, sizes_k=sizes[::-1])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [33, 48, 63, 64, 65, 96, 100, 127, 128])
@pytest.mark.parametrize("cap,axes", [(0.0, 0), (8.0, 3), (300.0, 1)])
def test_tiles_of_128_rows(dtype, d, cap, axes):
    x = ragged(d, dtype, d, axes)
    if not (dtype == "f32" and d > 64):
        assert (128, 1) in taken(x)
    got = compare(x, cap=cap)
    # rows of examples without rows on the other side
    for mine, other, names in (("q", "k", ("out", "dq")),
                               ("k", "q", ("dk", "dv"))):
        alone = ~torch.isin(x["batch_" + mine], x["batch_" + other])
        assert alone.any()
        for n in names:
            assert (got[n][alone] == 0).all(), n


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [48, 64, 128])
def test_tiles_of_128_rows_anywhere_in_memory(dtype, d):
    x = ragged(d, dtype, d, axes=2)
    want = call(x, cap=5.0)
    moved = {n: shifted(x[n]) for n in ("q", "k", "v", "dout")}
    got = call(dict(x, **moved), cap=5.0)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_tiles_of_128_rows_with_shared_key_heads(dtype, d):
    # (rows of q with two heads each: a tile ends between the two heads of none)
    x = ragged(d + 1, dtype, d, axes=1, heads=16)
    assert (128, 1) in taken(x) or (dtype == "f32" and d > 64)
    compare(x, cap=50.0)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_tiles_of_128_rows_keep_examples_apart(dtype, d, bad):
    x = ragged(d + 2, dtype, d, axes=3)
    want = call(x)
    some = (3, 20, 21, 40)
    inside = {s: sum(x["batch_" + s] == b for b in some) > 0 for s in "qk"}
    x = dict(x)
    for n, s in (("q", "q"), ("dout", "q"), ("k", "k"), ("v", "k")):
        x[n] = x[n].clone()
        x[n][inside[s]] = bad
    got = call(x)
    for n, s in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "k")):
        assert torch.equal(got[n][~inside[s]], want[n][~inside[s]]), n


# ---- sides cut into pieces --------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [5, 31, 65, 127])
@pytest.mark.parametrize("few,heads", CUT)
@pytest.mark.parametrize("side", ["q", "k"])
def test_pieces_of_odd_widths(dtype, d, few, heads, side):
    nq, nk = (few, 2300) if side == "q" else (2300, few)
    x = inputs(d + few, nq, nk, heads, heads, d, TYPES[dtype], axes=2)
    rows = 16 if few <= 256 else 64
    for p in range(3) if few > 256 else ((0, 1) if side == "q" else (2,)):
        got_rows, pieces = taken(x)[p]
        assert got_rows in (rows, 64) and pieces > 1, PASSES[p]
    compare(x, cap=20.0)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [31, 64])
def test_tiles_in_pieces_beside_whole_ones(dtype, d):
    # a long example, short ones and one without keys
    sizes_q, sizes_k = [1150, 40, 3, 90, 0], [1400, 30, 0, 700, 5]
    x = inputs(d, sum(sizes_q), sum(sizes_k), 4, 2, d, TYPES[dtype], axes=3,
               sizes_q=sizes_q, sizes_k=sizes_k)
    assert all(pieces > 1 for _, pieces in taken(x))
    compare(x)


# ---- what rounding takes off the output --------------------------------------------

def near_values(dtype, nq, nk, zero):
    """Even weights (powers of two, exact), values close to 8: the output is rounded by
    more than the values differ, in all rows' gradients alike."""
    g = torch.Generator().manual_seed(nq)
    x = inputs(nq, nq, nk, 4, 2, 64, TYPES[dtype])
    step = 8 * torch.finfo(TYPES[dtype]).eps
    x["v"] = (8 + step * torch.randint(0, 8, (nk, 2, 64), generator=g)) \
        .to(TYPES[dtype]).to(DEV)
    for n in "qk":
        x[n] = (1 + 0.25 * torch.rand(x[n].shape, generator=g)) \
            .to(TYPES[dtype]).to(DEV)
    x[zero] = torch.zeros_like(x[zero])
    return x


def backward(x, with_rest):
    """Gradients by the C ABI."""
    lib, (nq, hq, d), (nk, hk, _) = _native.capi, x["q"].shape, x["k"].shape
    codes = {torch.float32: 0, torch.float16: 2, torch.bfloat16: 3}
    args = _native.AttentionArgs(
        q=x["q"].data_ptr(), k=x["k"].data_ptr(), v=x["v"].data_ptr(),
        q_row=hq * d, q_head=d, k_row=hk * d, k_head=d, v_row=hk * d, v_head=d,
        dtype=codes[x["q"].dtype], nq=nq, nk=nk, hq=hq, hk=hk, d=d,
        scale=d ** -0.5, cap=0.0)
    out, dq = torch.empty_like(x["q"]), torch.empty_like(x["q"])
    rest = torch.empty_like(out) if with_rest else None
    dk, dv = torch.empty_like(x["k"]), torch.empty_like(x["v"])
    lse = torch.empty(hq, nq, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    for back in (0, 1):
        size = lib.pca_attention_workspace_bytes(nq, nk, hq, hk, d, back)
        room = torch.empty(size, dtype=torch.uint8, device=DEV)
        left = rest.data_ptr() if with_rest else None
        if back:
            rc = lib.pca_attention_backward(
                ctypes.byref(args), out.data_ptr(), left, lse.data_ptr(),
                x["dout"].data_ptr(), hq * d, d, dq.data_ptr(), dk.data_ptr(),
                dv.data_ptr(), room.data_ptr(), size, stream)
        else:
            rc = lib.pca_attention_forward(
                ctypes.byref(args), out.data_ptr(), left, lse.data_ptr(),
                room.data_ptr(), size, stream)
        assert rc == 0, lib.pca_last_error()
    torch.cuda.synchronize()
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("nq,nk", [(1, 256), (20, 1024), (300, 256),
                                   (600, 2048)])
@pytest.mark.parametrize("zero", ["q", "k"])
def test_gradients_do_not_see_the_output_rounded(dtype, nq, nk, zero):
    x = near_values(dtype, nq, nk, zero)
    got = call(x)
    val, err = attention_bounds(**x, exact_weights=True)
    check(got, val, err)
    again = backward(x, with_rest=True)
    for n in got:
        assert torch.equal(again[n], got[n]), n
    # without it they do, and are as near as that lets them be
    less = backward(x, with_rest=False)
    loose = attention_bounds(**x, exact_weights=True, rest=False)[1]
    check(less, val, loose)
    name = "dk" if zero == "q" else "dq"  # (sums of zeros)
    assert (less[name] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nq,nk", [(1, 256), (20, 1024), (300, 256),
                                   (600, 2048)])
def test_an_output_rounded_down_everywhere(dtype, nq, nk):
    # 7 of 16 values one step above 8: the output loses 0.44 of a step in every channel,
    # and a gradient of one sign adds that up.  What the gradients are off without
    # `rest` is beyond their bound with it.
    x = near_values(dtype, nq, nk, "q")
    g = torch.Generator().manual_seed(1)
    up = torch.rand(nk, 2, 64, generator=g).argsort(0) < nk * 7 // 16
    step = 8 * torch.finfo(TYPES[dtype]).eps
    x["v"] = (8 + step * up).to(TYPES[dtype]).to(DEV)
    x["dout"] = x["dout"].abs()
    got = call(x)
    val, err = attention_bounds(**x, exact_weights=True)
    check(got, val, err)
    less = backward(x, with_rest=False)
    check(less, val, attention_bounds(**x, exact_weights=True, rest=False)[1])
    off = (less["dq"].double() - val["dq"]).abs()
    assert (off > err["dq"]).double().mean() > 0.5
