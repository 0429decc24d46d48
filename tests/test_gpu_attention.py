"""attention against its definition in 64 bits: types, widths of heads, shared
heads, lengths from one row on, examples that share a tile, masks that leave a
row empty, strides, gradients, graphs, streams.
"""
import pytest
import torch

import pytorch_cluster_amd as pca
from features_common import attention64, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def inputs(seed, nq, nk, hq, hk, d, dtype, axes=0, sizes_q=None, sizes_k=None,
           dout=True):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(DEV)
    x = {"q": normal(nq, hq, d), "k": normal(nk, hk, d),
         "v": normal(nk, hk, d)}
    if sizes_q is not None:
        ids = torch.arange(len(sizes_q))
        x["batch_q"] = ids.repeat_interleave(torch.tensor(sizes_q)).to(DEV)
        x["batch_k"] = ids.repeat_interleave(torch.tensor(sizes_k)).to(DEV)
    if axes:
        x["pos_q"] = (3 * torch.rand(nq, axes, generator=g) + 10).to(DEV)
        x["pos_k"] = (3 * torch.rand(nk, axes, generator=g) + 10).to(DEV)
        x["slope"] = (2.0 ** -torch.arange(hq).float()).to(DEV)
    if dout:
        x["dout"] = normal(nq, hq, d)
    return x


def call(x, **more):
    """Entry point with gradients -> dict."""
    x = dict(x, **more)
    dout = x.pop("dout", None)
    if dout is None:
        return {"out": pca.attention(**x)}
    q, k, v = (x[n].detach().requires_grad_() for n in ("q", "k", "v"))
    out = pca.attention(**dict(x, q=q, k=k, v=v))
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def compare(x, **more):
    got = call(x, **more)
    val, err = attention64(**dict(x, **more))
    check(got, val, err)
    return got


# ---- one example --------------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (3, 17), (16, 16), (17, 33),
                                   (64, 64), (65, 63), (130, 200), (5, 1000),
                                   (700, 9)])
def test_lengths(dtype, nq, nk):
    compare(inputs(nq * 1000 + nk, nq, nk, 2, 2, 32, TYPES[dtype]))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [1, 5, 8, 16, 31, 40, 48, 64, 65, 80, 96, 127,
                               128])
def test_widths(dtype, d):
    compare(inputs(d, 50, 70, 2, 1, d, TYPES[dtype]))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 3), (6, 2), (8, 1), (7, 1)])
def test_heads(dtype, hq, hk):
    compare(inputs(hq * 10 + hk, 41, 77, hq, hk, 24, TYPES[dtype], axes=3))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("axes", [1, 2, 3])
@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_bias_and_cap(dtype, axes, cap):
    compare(inputs(axes, 90, 150, 4, 2, 64, TYPES[dtype], axes=axes), cap=cap)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [32, 64, 128])
def test_many_rows(dtype, d):
    # enough rows for the kernels that own 128 of them
    compare(inputs(d, 9000, 300, 4, 4, d, TYPES[dtype], axes=3), cap=20.0)
    compare(inputs(d + 1, 300, 9000, 4, 4, d, TYPES[dtype]))


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_one_query_over_many_rows(dtype):
    compare(inputs(1, 1, 20000, 8, 2, 128, TYPES[dtype], axes=1))


# ---- examples -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_examples_that_share_a_tile(dtype):
    sizes_q = [3, 1, 0, 40, 17, 16, 2, 5, 0, 64, 1]
    sizes_k = [5, 0, 7, 33, 1, 64, 31, 2, 0, 100, 3]
    x = inputs(7, sum(sizes_q), sum(sizes_k), 4, 2, 40, TYPES[dtype], axes=3,
               sizes_q=sizes_q, sizes_k=sizes_k)
    got = compare(x, cap=10.0)
    # rows of an example without keys
    alone = x["batch_q"] == 1
    assert (got["out"][alone] == 0).all() and (got["dq"][alone] == 0).all()
    # rows of an example without queries
    unseen = x["batch_k"] == 2
    assert (got["dk"][unseen] == 0).all() and (got["dv"][unseen] == 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("examples", [40, 700])
def test_many_small_examples(dtype, examples):
    g = torch.Generator().manual_seed(examples)
    sizes = torch.randint(0, 40, (examples,), generator=g).tolist()
    n = sum(sizes)
    x = inputs(examples, n, n, 4, 4, 32, TYPES[dtype], axes=2, sizes_q=sizes,
               sizes_k=sizes)
    x["batch_k"] = x["batch_q"]  # one tensor for both sides
    compare(x)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_one_query_per_example(dtype):
    sizes_k = [900, 1, 3000, 0, 64, 65, 128, 127, 2, 511] * 3
    x = inputs(5, 30, sum(sizes_k), 8, 2, 64, TYPES[dtype],
               sizes_q=[1] * 30, sizes_k=sizes_k)
    compare(x)


def test_batch_ids_with_gaps_and_int32():
    sizes = [10, 20, 30]
    x = inputs(3, 60, 60, 2, 2, 16, torch.float32, sizes_q=sizes,
               sizes_k=sizes)
    want = call(x)
    spread = torch.tensor([-5, 7, 2 ** 40], device=DEV)
    got = call(x, batch_q=spread[x["batch_q"]], batch_k=spread[x["batch_k"]])
    for n in want:
        assert torch.equal(got[n], want[n])
    got = call(x, batch_q=x["batch_q"].int(), batch_k=x["batch_k"].int())
    for n in want:
        assert torch.equal(got[n], want[n])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_of_other_examples_reach_nothing(dtype, bad):
    sizes_q, sizes_k = [5, 20, 9, 70], [30, 3, 50, 90]
    x = inputs(11, 104, 173, 2, 2, 32, TYPES[dtype], axes=3, sizes_q=sizes_q,
               sizes_k=sizes_k)
    want = call(x)
    inside_q, inside_k = x["batch_q"] == 1, x["batch_k"] == 1
    for n in ("q", "dout"):
        x[n] = x[n].clone()
        x[n][inside_q] = bad
    for n in ("k", "v"):
        x[n] = x[n].clone()
        x[n][inside_k] = bad
    x["pos_k"] = x["pos_k"].clone()
    x["pos_k"][inside_k] = bad
    got = call(x)
    for n, inside in (("out", inside_q), ("dq", inside_q), ("dk", inside_k),
                      ("dv", inside_k)):
        assert torch.equal(got[n][~inside], want[n][~inside]), n
        if bad != bad:
            assert not torch.isfinite(got[n][inside].float()).any(), n


@pytest.mark.parametrize("nq,nk", [(0, 5), (5, 0), (0, 0)])
def test_no_rows(nq, nk):
    x = inputs(1, nq, nk, 2, 2, 16, torch.bfloat16, axes=2,
               sizes_q=[nq, 0], sizes_k=[0, nk])
    got = call(x)
    for n in ("out", "dq"):
        assert got[n].shape == (nq, 2, 16) and (got[n] == 0).all()
    for n in ("dk", "dv"):
        assert got[n].shape == (nk, 2, 16) and (got[n] == 0).all()


# ---- values ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_large_scores(dtype):
    # sums whose maximum keeps growing along the keys, and one that dwarfs all
    x = inputs(2, 40, 600, 2, 2, 32, TYPES[dtype])
    x["k"] = (x["k"].float() * torch.linspace(0.1, 30, 600, device=DEV)
              .view(-1, 1, 1)).to(TYPES[dtype])
    compare(x)
    x["k"][599] = 100
    compare(x)


def test_scores_that_overflow():
    x = inputs(4, 20, 50, 1, 1, 16, torch.float32, dout=False)
    x["q"][3, 0, 0] = 3e38
    x["k"][:, 0, 0] = 0.5
    x["k"][7, 0, 0] = 3.0  # row 3: one score of +inf
    out = call(x, scale=1.0)["out"]
    assert torch.isnan(out[3]).all()
    keep = torch.arange(20, device=DEV) != 3
    assert torch.isfinite(out[keep]).all()


@pytest.mark.parametrize("nq, nk", [(1, 70), (3, 9000), (80, 50), (300, 9000)])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_scores_that_are_not_numbers(dtype, nq, nk):
    # all scores of a row, in every piece that its keys are cut into
    x = inputs(5, nq, nk, 1, 1, 32, TYPES[dtype], dout=False)
    x["q"][nq // 2, 0, 3] = float("nan")
    out = call(x)["out"]
    assert torch.isnan(out[nq // 2]).all()
    keep = torch.arange(nq, device=DEV) != nq // 2
    assert torch.isfinite(out[keep]).all()


def test_all_scores_minus_infinity():
    x = inputs(4, 20, 50, 1, 1, 16, torch.float32, axes=1, dout=False)
    x["pos_q"][3] = float("inf")
    out = call(x)["out"]
    assert (out[3] == 0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** 10])
def test_fp16_gradients_of_any_size(size):
    # gradients near the end of fp16's range keep its precision
    x = inputs(6, 200, 900, 2, 2, 64, torch.float16)
    x["dout"] = (x["dout"].float() * size).half()
    got = call(x)
    val, err = attention64(**x)
    check(got, val, err)


# ---- layouts --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [24, 32, 63])
def test_views_of_one_tensor(dtype, d):
    # q, k and v as slices of one projection, and heads before rows
    g = torch.Generator().manual_seed(d)
    qkv = torch.randn(80, 3, 4, d, generator=g).to(TYPES[dtype]).to(DEV)
    x = {"q": qkv[:, 0], "k": qkv[:, 1], "v": qkv[:, 2]}
    x["dout"] = torch.randn(80, 4, d, generator=g).to(TYPES[dtype]).to(DEV)
    want = call({n: t.contiguous() for n, t in x.items()})
    got = call(x)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    turned = {n: t.transpose(0, 1).contiguous().transpose(0, 1)
              for n, t in x.items()}
    got = call(turned)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    # last dimension not dense, and a base that is not on 16 bytes
    odd = {n: torch.empty(80, 4, 2 * d, dtype=TYPES[dtype],
                          device=DEV)[..., ::2].copy_(t)
           for n, t in x.items()}
    got = call(odd)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    shifted = {}
    for n, t in x.items():
        s = torch.empty(t.numel() + 1, dtype=TYPES[dtype], device=DEV)[1:]
        shifted[n] = s.view(t.shape).copy_(t)
    got = call(shifted)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("row", [4_000_000, 10_000_008])
def test_rows_far_apart(row):
    # offsets beyond 2^31 elements; tiles addressed by 32 bits and, where rows
    # are too far apart for that, by 64
    x = inputs(15, 30, 600, 2, 2, 64, torch.bfloat16, axes=1)
    want = call(x)
    room = torch.empty(600 * row + 128, dtype=torch.bfloat16, device=DEV)
    far = dict(x)
    for n, at in (("k", 0), ("v", row // 2)):
        far[n] = room[at:].as_strided((600, 2, 64), (row, 64, 1)) \
            .copy_(x[n])
    assert far["k"].storage_offset() + 599 * row > 2 ** 31
    got = call(far)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    # the same for the rows that dk and dv loop over
    want = call(dict(x, q=x["k"], k=x["q"], v=x["q"], dout=x["k"],
                     pos_q=x["pos_k"], pos_k=x["pos_q"]))
    got = call(dict(x, q=far["k"], k=x["q"], v=x["q"], dout=far["k"],
                    pos_q=x["pos_k"], pos_k=x["pos_q"]))
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_expanded_gradient():
    x = inputs(8, 30, 40, 2, 2, 32, torch.float32)
    q = x["q"].requires_grad_()
    pca.attention(q, x["k"], x["v"]).sum().backward()
    x["dout"] = torch.ones_like(q)
    assert torch.equal(q.grad, call(x)["dq"])


# ---- the call -------------------------------------------------------------------

@pytest.mark.parametrize("rows", [100, 3000])
def test_same_call_same_bits(rows):
    x = inputs(9, rows, rows, 4, 2, 64, torch.bfloat16, axes=3)
    first = call(x)
    for _ in range(3):
        again = call(x)
        for n in first:
            assert torch.equal(first[n], again[n]), n


def test_gradients_of_some_inputs():
    x = inputs(10, 40, 50, 2, 2, 32, torch.float32)
    want = call(x)
    v = x["v"].detach().requires_grad_()
    out = pca.attention(x["q"], x["k"], v)
    assert torch.equal(torch.autograd.grad(out, v, x["dout"])[0], want["dv"])
    out = pca.attention(x["q"], x["k"], v)
    assert out.requires_grad
    with torch.no_grad():
        assert not pca.attention(x["q"], x["k"], v).requires_grad


def test_no_second_derivative():
    x = inputs(10, 10, 10, 1, 1, 8, torch.float32)
    q = x["q"].requires_grad_()
    out = pca.attention(q, x["k"], x["v"])
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(out.sum(), q, create_graph=True)


def test_gradients_against_differences():
    # central differences of the definition in 64 bits, in random directions
    x = inputs(12, 12, 15, 2, 1, 8, torch.float32, axes=2)
    got = call(x, cap=3.0)
    g = torch.Generator().manual_seed(0)
    for name, grad in (("q", "dq"), ("k", "dk"), ("v", "dv")):
        step = torch.randn(x[name].shape, generator=g).double().to(DEV)
        h = 1e-5

        def value(sign):
            moved = dict(x)
            moved.pop("dout")
            moved[name] = x[name].double() + sign * h * step
            for other in ("q", "k", "v"):
                moved[other] = moved[other].double()
            val, _ = attention64(**moved, cap=3.0)
            return (val["out"] * x["dout"].double()).sum()
        want = (value(1) - value(-1)) / (2 * h)
        have = (got[grad].double() * step).sum()
        # h^2 of the third derivative and fp32's gradients: 1e-5 of the sum of
        # what is added up
        assert abs(want - have) <= 1e-5 * (got[grad].double() * step).abs().sum()


def test_on_another_stream():
    x = inputs(13, 500, 600, 4, 4, 64, torch.float16, axes=3,
               sizes_q=[200, 300], sizes_k=[100, 500])
    want = call(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(x)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("rows", [60, 2500])
def test_in_a_graph(rows):
    sizes = [rows // 3, rows - rows // 3]
    x = inputs(14, rows, rows, 4, 2, 64, torch.bfloat16, axes=3,
               sizes_q=sizes, sizes_k=sizes)
    leaves = {n: x[n].detach().clone().requires_grad_() for n in "qkv"}
    rest = {n: t for n, t in x.items() if n not in ("q", "k", "v", "dout")}

    def step():
        out = pca.attention(**leaves, **rest, cap=5.0)
        grads = torch.autograd.grad(out, tuple(leaves.values()), x["dout"])
        return (out.detach(),) + grads  # (no graph of the leaves stays)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(other):  # a second one with workspaces of its own
        held2 = step()
    for k in range(4):
        fresh = inputs(100 + k, rows, rows, 4, 2, 64, torch.bfloat16)
        with torch.no_grad():
            for n in "qkv":
                leaves[n].copy_(fresh[n])
        x["dout"].copy_(fresh["dout"])
        graph.replay()
        other.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b, c in zip(held, held2, want):
            assert torch.equal(a, c) and torch.equal(b, c), k
