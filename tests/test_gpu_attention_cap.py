"""attention with caps of every size: a large one bends nothing and costs no digits, a
tiny one leaves no score, in every type, forwards and backwards.
"""
import pytest
import torch

from attention_bounds import attention_bounds
from features_common import check
from test_gpu_attention import DEV, TYPES, call, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("nq,nk,d", [(60, 90, 32), (1, 700, 64), (90, 40, 128)])
@pytest.mark.parametrize("cap", [0.5, 100.0, 128.0, 129.0, 1e3, 1e4, 1e6, 1e9,
                                 1e38])
def test_caps_of_every_size(dtype, nq, nk, d, cap):
    x = inputs(nq, nq, nk, 4, 2, d, TYPES[dtype], axes=3)
    got = call(x, cap=cap)
    val, err = attention_bounds(**x, cap=cap)
    check(got, val, err)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("cap", [150.0, 1e4])
def test_scores_around_and_beyond_the_cap(dtype, cap):
    # products from far below the cap to some times it
    x = inputs(3, 50, 200, 2, 2, 32, TYPES[dtype])
    size = torch.logspace(-3, 0.6, 200, device=DEV).view(-1, 1, 1) * cap / 5
    x["k"] = (x["k"].float() * size).to(TYPES[dtype])
    got = call(x, cap=cap)
    val, err = attention_bounds(**x, cap=cap)
    check(got, val, err)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("cap", [1e39, 1e300])
def test_a_cap_beyond_fp32_bends_nothing(dtype, cap):
    x = inputs(4, 40, 60, 2, 1, 48, TYPES[dtype], axes=1)
    got = call(x, cap=cap)
    val, err = attention_bounds(**x, cap=cap)
    check(got, val, err)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("cap", [1e-20, 1e-37, 1e-42, 1e-300])
def test_a_tiny_cap_leaves_no_score(dtype, cap):
    # weights are even whatever the products are, zeros among them; the gradients of q
    # and k (1 - tanh^2 is 0 but for products of zero) stay finite
    x = inputs(5, 30, 64, 2, 2, 32, TYPES[dtype])
    x["q"][3] = 0
    got = call(x, cap=cap, scale=1.0)
    val, err = attention_bounds(**dict(x, q=torch.zeros_like(x["q"])),
                                exact_weights=True)
    for n in ("out", "dv"):
        check({n: got[n]}, val, err)
    for n in ("dq", "dk"):
        assert torch.isfinite(got[n]).all(), n
    some = torch.arange(30, device=DEV) != 3
    assert (got["dq"][some] == 0).all()
