"""lookup whose output has more than 2^31 pieces of 16 bytes: every row of it."""
import pytest
import torch

import pytorch_cluster_amd as pca

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype,width", [(torch.float32, 5), (torch.float16, 9),
                                         (torch.bfloat16, 9)])
def test_more_pieces_than_32_bits_count(dtype, width):
    # (two pieces a row, the second with one component)
    entries, table = 2 ** 30 + 777, 1000
    g = torch.Generator().manual_seed(width)
    weight = torch.randn(table, width, generator=g).to(dtype).to(DEV)
    index = torch.empty(entries, dtype=torch.int32, device=DEV)
    step = 1 << 26
    for at in range(0, entries, step):
        # (-1, and 1,000, name no row)
        e = torch.arange(at, min(at + step, entries), device=DEV)
        index[at:at + step] = (e * 7919 + (e >> 20)) % (table + 2) - 1
    out = pca.lookup(weight, index, 1.5)
    # one product in fp32, one rounding
    rows = torch.zeros(table + 2, width, dtype=dtype, device=DEV)
    rows[1:-1] = (weight.float() * 1.5).to(dtype)
    for at in range(0, entries, step):
        want = rows[index[at:at + step].long() + 1]
        assert torch.equal(out[at:at + step], want), at
