"""sample_rows over rows whose values lie further apart than the largest fp32 number: distances of 6e38 weigh what they
weigh at temperatures that are as large."""
import math

import pytest
import torch

from speech_serving import ops
from test_sample_rows_gpu import DEV, pick
from test_sample_rows_weights_gpu import borders

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1.0, 1e36, 5e37, 1e38, 3e38])
@pytest.mark.parametrize("dtype,n", [(torch.float32, 40), (torch.float32, 3000), (torch.bfloat16, 3000)])
def test_distances_beyond_the_largest_number(dtype, n, t):
    g = torch.Generator().manual_seed(n)
    x = (torch.rand(n, generator=g) * 2 - 1) * 3.2e38
    x[n // 3] = 3.3e38
    x = x.to(dtype)
    assert torch.isinf(x.max() - x.float()).any() and torch.isfinite(x).all()
    temperature = float(torch.tensor(t, dtype=torch.float32))
    w = ((x.double() - x.double().max()) / temperature).exp()
    u = torch.rand(20, generator=g)
    if t > 1e37:
        u = torch.cat((u, borders(w.cumsum(0), 10, n)))
    rows = x.expand(len(u), n).contiguous()
    for k, p, least in ((0, 1.0, 0.0), (10, 1.0, 0.0), (0, 0.6, 0.0), (0, 0.95, 0.0), (n // 2, 0.9, 0.0), (0, 1.0, 0.05)):
        got = ops.sample_rows(rows.to(DEV), u.to(DEV), t, k, p, least)
        assert got.tolist() == [pick(x, v, t, k, p, least) for v in u]


def test_an_infinite_temperature():
    x = torch.tensor([3e38, -3e38, 0.0, -1e38, 3e38, -math.inf]).repeat(10, 1)
    for k, want in ((0, [2, 2, 2, 2, 2]), (4, [2, 0, 3, 2, 3]), (2, [5, 0, 0, 0, 5])):
        got = ops.sample_rows(x.to(DEV), ((torch.arange(10) + 0.5) / 10).to(DEV), math.inf, k)
        assert got.bincount(minlength=5).tolist() == want
