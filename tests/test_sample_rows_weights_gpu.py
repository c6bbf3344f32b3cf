"""sample_rows where a random number, or top-p, lies as near as fp32 numbers can to a border between two columns: one
large value, and columns so small beside it that their distance from it does not fit in 32 bits."""
import pytest
import torch

from test_sample_rows_gpu import check

pytestmark = pytest.mark.gpu


def borders(cum, count, seed):
    """fp32 numbers on both sides of cum[j] / cum[-1] for some j, [2 * count], as near as multiples of 2^-24 come; those
    nearer than 2^-28 (weights in units of 2^-44 would have a say) are passed over."""
    share = cum / cum[-1]
    below = (share * 2.0 ** 24).floor() * 2.0 ** -24
    fine = (share - below > 2.0 ** -28) & (below + 2.0 ** -24 - share > 2.0 ** -28) & (share < 0.999)
    fine = fine.nonzero()[:, 0]
    j = fine[torch.randperm(len(fine), generator=torch.Generator().manual_seed(seed))[:count]]
    assert len(j) == count
    return torch.cat((below[j], below[j] + 2.0 ** -24)).float()


ROWS = [  # type, largest value, size of the others, temperature, columns
    (torch.bfloat16, 8.0, 1.97887421e-05, 1.0, 3001),
    (torch.bfloat16, 8.625, 3e-6, 1.0, 6000),
    (torch.bfloat16, 100.0, 1e-3, 12.0, 3001),
    (torch.float16, 8.625, 2e-5, 1.0, 3001),
    (torch.float16, 11.0, 1e-4, 1.4, 20000),
    (torch.float16, 5.5, 1e-5, 0.7, 400),
    (torch.bfloat16, 5.5, 1e-5, 0.7, 400),
    (torch.float32, 8.625, 2e-5, 1.0, 3001),
]


@pytest.mark.parametrize("alike", [True, False])
@pytest.mark.parametrize("dtype,top,size,t,n", ROWS)
def test_borders_between_small_columns(dtype, top, size, t, n, alike):
    g = torch.Generator().manual_seed(n)
    x = torch.full((n,), size) if alike else torch.randn(n, generator=g) * size
    x[0] = top
    x = x.to(dtype)
    temperature = float(torch.tensor(t, dtype=torch.float32))
    w = ((x.double() - top) / temperature).exp()
    u = borders(w.cumsum(0), 40, n)
    check(x.expand(80, n).contiguous(), u, t)
    # the columns before which less than p of the weight lies, in the order of their values; the last by place is drawn
    p = borders(w[torch.argsort(-x.double(), stable=True)].cumsum(0), 40, n + 1)
    check(x.expand(80, n).contiguous(), torch.full((80,), 1.0 - 2.0 ** -24), t, 0, p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("top,t,n", [(8.0, 1.0, 20001), (4.0, 0.7, 3001), (8.0, 1.0, 200001), (16.0, 2.0, 50001)])
def test_borders_between_columns_whose_distances_round_apart(dtype, top, t, n):
    """x - top of the first half lies half a step above what 32 bits hold, of the second half below (ties go to the same
    number): taken as they round, the halves' weights are off by 2^-24 top / t in both directions."""
    step = top * 2.0 ** -24
    x = torch.full((n,), 41.5 * step)
    x[n // 2 :] = 42.5 * step
    x[0] = top
    x = x.to(dtype)
    assert float(x[1]) == 41.5 * step and float(x[-1]) == 42.5 * step
    temperature = float(torch.tensor(t, dtype=torch.float32))
    w = ((x.double() - top) / temperature).exp()
    check(x.expand(80, n).contiguous(), borders(w.cumsum(0), 40, n), t)
    p = borders(w[torch.argsort(-x.double(), stable=True)].cumsum(0), 40, n + 1)
    check(x.expand(80, n).contiguous(), torch.full((80,), 1.0 - 2.0 ** -24), t, 0, p)
