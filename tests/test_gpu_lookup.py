"""lookup and the gradient of its table against their definition in 64 bits."""
import pytest
import torch

import pytorch_cluster_amd as pca
from features_common import check, lookup64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def inputs(seed, table, entries, width, dtype, skew=1.0, none=0.0):
    g = torch.Generator().manual_seed(seed)
    weight = torch.randn(table, width, generator=g).to(dtype).to(DEV)
    u = torch.rand(entries, generator=g).double()
    index = (u ** skew * table).long().clamp(max=max(table - 1, 0))
    if none:
        index[torch.rand(entries, generator=g) < none] = -1
    dout = torch.randn(entries, width, generator=g).to(dtype).to(DEV)
    return weight, index.to(DEV), dout


def call(weight, index, dout, scale):
    w = weight.detach().requires_grad_()
    out = pca.lookup(w, index, scale)
    return {"out": out, "dweight": torch.autograd.grad(out, w, dout)[0]}


def compare(weight, index, dout, scale=1.5):
    got = call(weight, index, dout, scale)
    val, err = lookup64(weight, index, scale, dout)
    check(got, val, err)
    with torch.no_grad():
        assert torch.equal(pca.lookup(weight, index, scale), got["out"])
    return got


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("table,entries", [
    (1, 1), (1, 5000), (3, 2), (255, 4096), (256, 4097), (257, 8192),
    (1000, 20000), (65535, 30000), (65536, 30000), (70000, 100),
    (100000, 300000)])
def test_sizes(dtype, table, entries):
    compare(*inputs(table + entries, table, entries, 16, TYPES[dtype]))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 20, 33, 64, 100, 128, 250,
                                   256, 300, 513, 1024])
def test_widths(dtype, width):
    compare(*inputs(width, 50, 5000, width, TYPES[dtype]))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("skew", [4.0, 40.0])
def test_few_rows_have_most_entries(dtype, skew):
    compare(*inputs(1, 4096, 200000, 24, TYPES[dtype], skew=skew))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("width", [5, 300, 1000])
def test_long_runs_of_wide_rows(dtype, width):
    # workgroups inside one run, in several columns, the last one in part
    compare(*inputs(8, 40, 30000, width, TYPES[dtype], skew=6.0, none=0.1))


def test_all_entries_in_one_row():
    weight, index, dout = inputs(2, 1000, 100000, 32, torch.bfloat16)
    for row in (0, 517, 999):
        compare(weight, torch.full_like(index, row), dout)


@pytest.mark.parametrize("entries", [300, 50000])
def test_entries_without_a_row(entries):
    weight, index, dout = inputs(3, 700, entries, 40, torch.float32, none=0.3)
    index[5] = 700
    index[6] = 2 ** 40
    index[7] = -2 ** 40
    got = compare(weight, index, dout)
    assert (got["out"][5:8] == 0).all()
    got = compare(weight, torch.full_like(index, -1), dout)
    assert (got["dweight"] == 0).all()


def test_values_of_entries_without_a_row_reach_nothing():
    weight, index, dout = inputs(3, 70, 3000, 8, torch.float32, none=0.3)
    want = call(weight, index, dout, 1.0)
    dout[index < 0] = float("nan")
    got = call(weight, index, dout, 1.0)
    assert torch.equal(got["dweight"], want["dweight"])


@pytest.mark.parametrize("table,entries", [(0, 5), (5, 0), (0, 0)])
def test_no_rows(table, entries):
    weight, index, dout = inputs(4, table, entries, 8, torch.float16)
    got = call(weight, index, dout, 1.0)
    assert got["out"].shape == (entries, 8) and (got["out"] == 0).all()
    assert got["dweight"].shape == (table, 8) and (got["dweight"] == 0).all()


def test_shapes_types_and_strides_of_the_index():
    weight, index, dout = inputs(5, 100, 600, 12, torch.float32)
    want = call(weight, index, dout, 2.0)
    got = call(weight, index.int(), dout, 2.0)
    assert torch.equal(got["out"], want["out"])
    assert torch.equal(got["dweight"], want["dweight"])
    table = index.view(30, 20)
    got = call(weight, table, dout.view(30, 20, 12), 2.0)
    assert torch.equal(got["out"], want["out"].view(30, 20, 12))
    assert torch.equal(got["dweight"], want["dweight"])
    got = call(weight, table.t(), dout.view(30, 20, 12).transpose(0, 1), 2.0)
    assert torch.equal(got["out"],
                       want["out"].view(30, 20, 12).transpose(0, 1))
    got = call(weight, index[7], dout[7], 2.0)
    assert got["out"].shape == (12,)
    # a column of a wider table, a base that is not on 16 bytes
    wide = torch.randn(100, 25, device=DEV)
    wide[:, 1:13] = weight
    got = call(wide[:, 1:13], index, dout, 2.0)
    assert torch.equal(got["out"], want["out"])


def test_tables_beyond_2_to_the_31():
    # elements of the table, and pieces of 16 bytes of the output
    rows, width = 18_000_000, 128
    weight = torch.zeros(rows, width, dtype=torch.float16, device=DEV)
    g = torch.Generator().manual_seed(8)
    index = torch.randint(0, rows, (5000,), generator=g)
    index[:3] = torch.tensor([rows - 1, 0, rows - 1])
    index = index.to(DEV)
    weight[index] = torch.randn(5000, width, generator=g).half().to(DEV)
    weight.requires_grad_()
    out = pca.lookup(weight, index, 2.0)
    assert torch.equal(out, weight.detach()[index] * 2)
    dout = torch.randn(5000, width, generator=g).half().to(DEV)
    grad, = torch.autograd.grad(out, weight, dout)
    assert grad.shape == weight.shape
    few, place = torch.unique(index, return_inverse=True)
    val, err = lookup64(torch.zeros(len(few), width, dtype=torch.float16,
                                    device=DEV), place, 2.0, dout)
    check({"dweight": grad[few]}, val, err)
    grad[few] = 0
    assert not grad.any()


def test_expanded_gradient():
    weight, index, _ = inputs(5, 100, 600, 12, torch.float32)
    w = weight.requires_grad_()
    pca.lookup(w, index).sum().backward()
    count = torch.bincount(index, minlength=100).float()
    assert torch.equal(w.grad, count[:, None].expand(100, 12))


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_same_call_same_bits(dtype):
    x = inputs(6, 900, 150000, 32, TYPES[dtype], skew=3.0)
    first = call(*x, 0.5)
    for _ in range(3):
        assert torch.equal(first["dweight"], call(*x, 0.5)["dweight"])


def test_no_second_derivative():
    weight, index, dout = inputs(6, 9, 15, 3, torch.float32)
    w = weight.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(pca.lookup(w, index).sum(), w, create_graph=True)


@pytest.mark.parametrize("entries", [500, 60000])
def test_in_a_graph_and_on_another_stream(entries):
    weight, index, dout = inputs(7, 3000, entries, 64, torch.bfloat16)
    w = weight.detach().clone().requires_grad_()

    def step():
        out = pca.lookup(w, index, 2.0)
        grads = torch.autograd.grad(out, w, dout)
        return (out.detach(),) + grads  # (no graph of the leaf stays)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        _, fresh, fresh_dout = inputs(30 + k, 3000, entries, 64, torch.bfloat16)
        index.copy_(fresh)
        dout.copy_(fresh_dout)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), k
