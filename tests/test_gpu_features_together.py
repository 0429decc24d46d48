"""The operators on the rows' features as a layer uses them, next to the
searches: sampled rows (fps) of a batch of clouds look at all rows of their
cloud (norm_rotate, attention) and hand what they found to the nearest rows
(nearest, lookup).  Against the same layer in 64 bits on the same rows, and from
two streams and two threads at once.
"""
import threading

import pytest
import torch

import pytorch_cluster_amd as pca
from features_common import attention64, lookup64, norm_rotate64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = [300, 1, 777, 64]
HEADS, KV_HEADS, D = 4, 2, 32


def layer_inputs(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    n = sum(SIZES)

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(DEV)
    return {
        "pos": torch.rand(n, 3, generator=g).to(DEV),
        "batch": torch.arange(len(SIZES)).repeat_interleave(
            torch.tensor(SIZES)).to(DEV),
        "x": normal(n, HEADS * D),
        "kv": normal(n, KV_HEADS, 2 * D),
        "gain": normal(D),
        "freq": (6.0 * torch.rand(3, D // 2, generator=g)).to(DEV),
        "slope": torch.tensor([4.0, 1.0, 0.5, 0.1], device=DEV),
        "dout": normal(n, HEADS * D)}


def layer(c, x, kv, gain):
    """Rows for every row, and the row numbers on the way."""
    picked = pca.fps(c["pos"], c["batch"], 0.25, random_start=False)
    pos_q, batch_q = c["pos"][picked], c["batch"][picked]
    q = pca.lookup(x, picked).view(-1, HEADS, D)
    q, _ = pca.norm_rotate(q, None, pos_q, c["freq"], gain)
    k, _ = pca.norm_rotate(kv[..., :D], None, c["pos"], c["freq"], gain)
    found = pca.attention(q, k, kv[..., D:], batch_q, c["batch"], pos_q,
                          c["pos"], c["slope"], cap=8.0)
    near = pca.nearest(c["pos"], pos_q, c["batch"], batch_q)
    return pca.lookup(found.flatten(1), near, 0.5), picked, near


def gradients(c):
    leaves = [c[n].detach().requires_grad_() for n in ("x", "kv", "gain")]
    out, picked, near = layer(c, *leaves)
    return (out.detach(),) + torch.autograd.grad(out, leaves, c["dout"]), \
        picked, near


def layer64(c, picked, near):
    """The same, operator by operator, forwards and then backwards."""
    pos_q, batch_q = c["pos"][picked], c["batch"][picked]
    x, kv, gain, dout = (c[n].double() for n in ("x", "kv", "gain", "dout"))
    at = {"batch_q": batch_q, "batch_k": c["batch"], "pos_q": pos_q,
          "pos_k": c["pos"], "slope": c["slope"], "cap": 8.0}
    rows_q = x[picked].view(-1, HEADS, D)
    rows_k, v = kv[..., :D], kv[..., D:]
    q = norm_rotate64(rows_q, pos_q, c["freq"], gain)[0]["out"]
    k = norm_rotate64(rows_k, c["pos"], c["freq"], gain)[0]["out"]
    found = attention64(q, k, v, **at)[0]["out"]
    out = lookup64(found.flatten(1), near, 0.5)[0]["out"]
    dfound = lookup64(found.flatten(1), near, 0.5, dout)[0]["dweight"]
    g = attention64(q, k, v, dout=dfound.view(found.shape), **at)[0]
    gq = norm_rotate64(rows_q, pos_q, c["freq"], gain, 1e-6, g["dq"])[0]
    gk = norm_rotate64(rows_k, c["pos"], c["freq"], gain, 1e-6, g["dk"])[0]
    dx = lookup64(x, picked, 1.0, gq["dx"].flatten(1))[0]["dweight"]
    return (out, dx, torch.cat([gk["dx"], g["dv"]], -1),
            gq["dweight"] + gk["dweight"])


def test_a_layer_and_its_gradients():
    c = layer_inputs(0)
    got, picked, near = gradients(c)
    want = layer64(c, picked, near)
    for name, a, b in zip(("out", "dx", "dkv", "dgain"), got, want):
        assert a.shape == b.shape, name
        # Some thousand fp32 roundings (2^-24) on the way of a value, of numbers
        # that are at most some ten times the result's norm per row: 1e-3 of
        # the largest would be a mistake, 1e-4 bounds 1,600 roundings that all
        # point the same way.
        assert (a.double() - b).abs().max() <= 1e-4 * b.abs().max(), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_layer_in_16_bits_is_near_the_one_in_32(dtype):
    c = layer_inputs(1, dtype)
    got, picked, near = gradients(c)
    want = layer64(c, picked, near)
    # four operators, each off by a few half steps of values of its own size,
    # forwards and backwards: 32 half steps of the norm
    bound = 32 * torch.finfo(dtype).eps / 2
    for name, a, b in zip(("out", "dx", "dkv", "dgain"), got, want):
        assert (a.double() - b).norm() <= bound * b.norm(), name


def test_two_streams_and_threads_at_once():
    inputs = [layer_inputs(10 + i, torch.bfloat16) for i in range(2)]
    want = [gradients(c)[0] for c in inputs]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[i] = gradients(inputs[i])[0]
            stream.synchronize()
        except BaseException as e:  # noqa: B902  (told by the main thread)
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
