"""norm_rotate against its definition in 64 bits."""
import pytest
import torch

import pytorch_cluster_amd as pca
from features_common import check, norm_rotate64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def inputs(seed, rows, hq, hk, d, axes, rotated, dtype, weights=True,
           weight_dtype=None, reach=50.0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(DEV)
    x = {"q": normal(rows, hq, d), "k": normal(rows, hk, d) if hk else None,
         "pos": ((2 * torch.rand(rows, axes, generator=g) - 1) * reach).to(DEV),
         "freq": (100 * torch.rand(axes, rotated, generator=g)).to(DEV)}
    if weights:
        kind = weight_dtype or dtype
        x["weight_q"] = (1 + 0.2 * torch.randn(d, generator=g)).to(kind).to(DEV)
        if hk:
            x["weight_k"] = (1 + 0.2 * torch.randn(d, generator=g)) \
                .to(kind).to(DEV)
    return x, normal(rows, hq, d), normal(rows, hk, d) if hk else None


def compare(x, dq, dk, eps=1e-6):
    leaves = {n: x[n].detach().requires_grad_()
              for n in ("q", "k", "weight_q", "weight_k")
              if x.get(n) is not None}
    q, k = pca.norm_rotate(**dict(x, **leaves), eps=eps)
    outs, douts = (q, k), (dq, dk)
    if k is None:
        outs, douts = (q,), (dq,)
    grads = dict(zip(leaves, torch.autograd.grad(outs, tuple(leaves.values()),
                                                 douts)))
    for side, out, dout in zip("qk", outs, douts):
        weight = x.get("weight_" + side)
        val, err = norm_rotate64(x[side], x["pos"], x["freq"], weight, eps, dout)
        got = {"out": out, "dx": grads[side]}
        if weight is not None:
            got["dweight"] = grads["weight_" + side]
        check(got, val, err, side)
    with torch.no_grad():
        again, _ = pca.norm_rotate(**x, eps=eps)
    assert torch.equal(again, q)
    return q, k, grads


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows", [1, 2, 63, 1000, 9000])
def test_rows(dtype, rows):
    compare(*inputs(rows, rows, 4, 2, 64, 3, 30, TYPES[dtype]))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d,rotated", [(1, 0), (2, 1), (5, 2), (8, 4), (15, 1),
                                       (16, 8), (33, 16), (48, 21), (64, 32),
                                       (80, 40), (127, 63), (128, 63),
                                       (130, 65), (200, 99), (256, 128),
                                       (255, 127)])
def test_widths(dtype, d, rotated):
    compare(*inputs(d, 37, 3, 2, d, 2, rotated, TYPES[dtype]))


@pytest.mark.parametrize("hq,hk", [(1, 0), (1, 1), (8, 1), (3, 5), (32, 8)])
def test_heads(hq, hk):
    compare(*inputs(hq, 100, hq, hk, 32, 1, 16, torch.bfloat16))


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_weights(dtype):
    compare(*inputs(1, 50, 2, 2, 40, 3, 20, TYPES[dtype], weights=False))
    compare(*inputs(2, 50, 2, 2, 40, 3, 20, TYPES[dtype],
                    weight_dtype=torch.float32))
    x, dq, dk = inputs(3, 50, 2, 2, 40, 3, 20, TYPES[dtype])
    del x["weight_q"]
    compare(x, dq, dk)


def test_far_positions():
    # 10 km at 100 rad / m: the angle is known to a third of a turn in fp32
    compare(*inputs(4, 200, 2, 2, 64, 3, 32, torch.float32, reach=1e4))


def test_rows_of_zeros():
    x, dq, dk = inputs(5, 20, 2, 2, 32, 2, 16, torch.float32)
    x["q"][3] = 0
    compare(x, dq, dk, eps=1e-3)
    q, _ = pca.norm_rotate(**x)
    assert (q[3] == 0).all()


def test_no_rows():
    x, dq, dk = inputs(5, 0, 2, 2, 32, 2, 16, torch.float32)
    _, _, grads = compare(x, dq, dk)
    assert (grads["weight_q"] == 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [24, 32, 63])
def test_views_of_one_tensor(dtype, d):
    x, dq, dk = inputs(6, 50, 4, 4, d, 3, d // 2, TYPES[dtype])
    want = compare(x, dq, dk)
    both = torch.stack([x["q"], x["k"]], 1)
    got = compare(dict(x, q=both[:, 0], k=both[:, 1]), dq, dk)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for n in want[2]:
        assert torch.equal(got[2][n], want[2][n]), n
    flip = {n: x[n].transpose(0, 1).contiguous().transpose(0, 1) for n in "qk"}
    got = compare(dict(x, **flip), dq, dk)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_unused_output_and_second_derivative():
    x, dq, _ = inputs(7, 30, 2, 2, 32, 3, 16, torch.float32)
    k = x["k"].requires_grad_()
    q = x["q"].requires_grad_()
    out, _ = pca.norm_rotate(**x)
    gq, gk = torch.autograd.grad(out, (q, k), dq, allow_unused=True)
    val, err = norm_rotate64(q.detach(), x["pos"], x["freq"], x["weight_q"],
                             1e-6, dq)
    check({"dx": gq}, val, err)
    assert gk is None or (gk == 0).all()
    out, _ = pca.norm_rotate(**x)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(out.sum(), q, create_graph=True)


def test_in_a_graph_and_on_another_stream():
    x, dq, dk = inputs(8, 700, 4, 2, 64, 3, 32, torch.bfloat16)
    leaves = {n: x[n].detach().clone().requires_grad_()
              for n in ("q", "k", "weight_q", "weight_k")}

    def step():
        outs = pca.norm_rotate(**dict(x, **leaves))
        grads = torch.autograd.grad(outs, tuple(leaves.values()), (dq, dk))
        # (no graph of the leaves stays)
        return tuple(t.detach() for t in outs) + grads
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
        fresh, _, _ = inputs(20 + k, 700, 4, 2, 64, 3, 32, torch.bfloat16)
        with torch.no_grad():
            for n in leaves:
                leaves[n].copy_(fresh[n])
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), k
