"""attention of rows in which one key outweighs all others together: what a hundred
thousand small weights add up to is neither lost nor doubled.
"""
import pytest
import torch

from attention_bounds import attention_bounds
from features_common import check
from test_gpu_attention import DEV, TYPES, call, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("nq,nk", [(1, 200000), (40, 100000), (700, 20000)])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("below", [16.5, 17.375, 17.40625, 18.0])
def test_small_weights_add_up(dtype, nq, nk, place, below):
    # (17.4 is 25.1 in units of log 2: half of fp16's smallest number)
    x = inputs(1, nq, nk, 1, 1, 16, TYPES[dtype], dout=False)
    at = {"first": 0, "middle": nk // 2, "last": nk - 1}[place]
    x["q"].zero_()
    x["q"][:, 0, 0] = 1
    x["k"].zero_()
    x["k"][:, 0, 0] = -below
    x["k"][at] = 0
    x["v"] = x["v"].abs()
    x["v"][at] = 0
    got = call(x, scale=1.0)
    val, err = attention_bounds(**x, scale=1.0)
    check(got, val, err)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_gradients_of_small_weights(dtype):
    x = inputs(2, 30, 50000, 2, 1, 32, TYPES[dtype])
    x["k"][7] = 40 * x["q"][:, 0].mean(0)
    x["k"][20000] = 30
    got = call(x)
    val, err = attention_bounds(**x)
    check(got, val, err)
