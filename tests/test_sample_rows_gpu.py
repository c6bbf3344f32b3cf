"""sample_rows against its definition in 64 bits, row by row on the CPU.  Tokens have to be equal; log-probabilities are
within 2e-6 + 1e-6 |value| (a sum of n positive fp32 terms, each off by a few 2^-23, added in groups, and a logarithm)."""
import math

import pytest
import torch

from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pick(x, u, t=1.0, k=0, p=1.0, least=0.0):
    """One row in fp64; fp32 settings as they are stored."""
    x = x.double()
    t, p, least, u = (float(torch.tensor(float(s), dtype=torch.float32)) for s in (t, p, least, u))
    nan = torch.isnan(x)
    if nan.any():
        return int(nan.nonzero()[0])
    m = x.max()
    top = int((x == m).nonzero()[0])
    if not t > 0 or not torch.isfinite(m):
        return top
    order = torch.argsort(-x, stable=True)
    if k > 0:
        order = order[:k]
    w = torch.exp((x[order] - m) / t)
    if p < 1:
        before = torch.cat((w.new_zeros(1), w.cumsum(0)[:-1]))
        order = order[: max(1, int((before < p * w.sum()).sum()))]
    if least > 0:
        order = order[: max(1, int((x[order] >= m + t * math.log(least)).sum()))]
    left = order.sort().values
    cum = torch.exp((x[left] - m) / t).cumsum(0)
    at = int((cum <= max(0.0, u) * cum[-1]).sum())
    return int(left[min(at, len(left) - 1)])


def check(x, u, t=1.0, k=0, p=1.0, least=0.0, skip=None, cols=None, dev=None):
    rows, n = x.shape[0], cols or x.shape[1]

    def per_row(s, dtype):
        return s.to(DEV, dtype) if isinstance(s, torch.Tensor) else s

    logs = torch.full((rows,), 7.0, device=DEV)
    got = ops.sample_rows(x.to(DEV) if dev is None else dev, u.to(DEV), per_row(t, torch.float32), per_row(k, torch.int32),
                          per_row(p, torch.float32), per_row(least, torch.float32), cols=cols,
                          skip=None if skip is None else skip.to(DEV), logprobs=logs)
    y = x[:, :n].float()
    if skip is not None:
        y = y.masked_fill(skip[:n], -math.inf)
    of = lambda s, r: float(s[r]) if isinstance(s, torch.Tensor) else s  # noqa: E731
    want = [pick(y[r], u[r], of(t, r), int(of(k, r)), of(p, r), of(least, r)) for r in range(rows)]
    assert got.tolist() == want
    exact = torch.log_softmax(y.double(), -1)[torch.arange(rows), torch.tensor(want)]
    fine = torch.isfinite(exact)
    off = (logs.cpu().double() - exact).abs()
    assert (off[fine] <= 2e-6 + 1e-6 * exact[fine].abs()).all(), off[fine].max()
    assert not torch.isfinite(logs.cpu()[~fine]).any()
    return got


def rows_of(seed, rows, cols, spread=2.0, dtype=torch.float32, peaks=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * spread
    if peaks:
        x.scatter_add_(1, torch.randint(cols, (rows, 30), generator=g), torch.rand(rows, 30, generator=g) * torch.rand(rows, 1, generator=g) * 15)
    return x.to(dtype), torch.rand(rows, generator=g), g


@pytest.mark.parametrize("cols", [1, 2, 31, 257, 1000, 4096, 51865, 131073])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_settings_by_row(cols, dtype):
    rows = 24
    x, u, g = rows_of(cols, rows, cols, dtype=dtype)
    t = torch.rand(rows, generator=g) + 0.3
    t[3] = 0.0
    k = torch.randint(0, min(cols, 200) + 1, (rows,), generator=g) * (torch.rand(rows, generator=g) < 0.5)
    p = torch.where(torch.rand(rows, generator=g) < 0.6, torch.rand(rows, generator=g), torch.ones(rows))
    least = torch.where(torch.rand(rows, generator=g) < 0.3, torch.rand(rows, generator=g) * 0.3, torch.zeros(rows))
    check(x, u, t, k, p, least)


@pytest.mark.parametrize("rows", [1, 5, 160, 700])
def test_numbers_of_rows(rows):
    x, u, _ = rows_of(rows, rows, 6000, dtype=torch.bfloat16)
    check(x, u, 0.8, 50, 0.9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_rows_where_neighbours_weigh_alike(dtype):
    """A hundred thousand columns of nearly one weight: the sums' boundaries lie as close as they can."""
    x, u, _ = rows_of(1, 40, 100000, spread=0.5, dtype=dtype, peaks=False)
    check(x, u, 1.0)
    check(x, u, 1.3, 0, 0.9)


def test_ties():
    """Few distinct values: cuts fall among equal columns, which count by their place."""
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-3, 4, (60, 3000), generator=g).float() * 0.25
    u = torch.rand(60, generator=g)
    k = torch.randint(1, 3000, (60,), generator=g)
    check(x, u, 1.0, k)
    check(x, u, 1.0, 0, torch.rand(60, generator=g))
    check(x, u, 0.7, k, torch.rand(60, generator=g), torch.rand(60, generator=g) * 0.8)
    check(torch.zeros(9, 500), torch.rand(9, generator=g), 1.0, 100, 0.5)


def test_signed_zeros_are_one_value():
    x = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0]]).repeat(20, 1)
    check(x, torch.arange(20) / 20.0, 1.0, 2)
    check(x, torch.arange(20) / 20.0, 1.0, 0, 0.5)


@pytest.mark.parametrize("u", [0.0, 0.5, 1.0 - 2.0 ** -24])
def test_ends_of_the_random_number(u):
    x, _, _ = rows_of(3, 12, 5000)
    check(x, torch.full((12,), u), 1.0, 40, 0.95)
    check(x, torch.full((12,), u), 1.0)


def test_extreme_settings():
    x, u, _ = rows_of(4, 8, 3000)
    for t, k, p, least in ((1e-4, 0, 0.9, 0.0), (1e4, 0, 0.9, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 2999, 0.999, 0.0), (1.0, 5000, 0.5, 0.0),
                           (1.0, 0, 0.0, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 2.0), (1.0, -4, 2.0, -1.0),
                           (-1.0, 10, 0.5, 0.1), (float("nan"), 10, 0.5, 0.1), (1.0, 0, 1.0 - 2.0 ** -24, 0.0), (0.05, 400, 0.7, 1e-6)):
        check(x, u, t, k, p, least)


def test_wide_values():
    """Values over the whole range of fp32, and of each 16-bit type."""
    g = torch.Generator().manual_seed(5)
    for dtype, top in ((torch.float32, 80), (torch.bfloat16, 80), (torch.float16, 9)):
        x = (torch.randn(12, 4000, generator=g) * torch.exp(torch.rand(12, 4000, generator=g) * top - top / 2)).to(dtype)
        check(x, torch.rand(12, generator=g), 1.0, torch.randint(0, 4000, (12,), generator=g), 0.9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_not_finite_values_and_masks(dtype):
    x, u, _ = rows_of(6, 8, 700, dtype=dtype)
    x[0, 300], x[0, 400] = math.nan, math.inf
    x[1, 5], x[1, 600] = math.inf, math.inf
    x[2, :] = -math.inf
    x[3, 1:] = -math.inf
    x[4, 100:650] = -math.inf
    x[5, :] = torch.finfo(dtype).min
    check(x, u, 1.0, 0, 0.9)
    check(x, u, 1.0, 20)
    skip = torch.zeros(700, dtype=torch.bool)
    skip[::3] = True
    check(x, u, 0.9, 30, 0.9, 0.01, skip=skip)
    check(x, u, 1.0, skip=torch.ones(700, dtype=torch.bool))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strided_rows(dtype):
    """Rows off 16-byte boundaries, fewer columns than a row holds, and a mask off its boundary."""
    wide, u, _ = rows_of(7, 10, 5005, dtype=dtype)
    wide = wide.to(DEV)
    for lo, cols in ((0, 5001), (1, 4999), (3, 16), (8, 4990)):
        view = wide[:, lo:]
        skip = torch.zeros(5006, dtype=torch.bool, device=DEV)[lo : lo + cols]
        skip[::7] = True
        check(view.cpu(), u, 0.9, 60, 0.95, cols=cols, skip=skip.cpu(), dev=view)


def test_order_of_rows_and_graphs_change_nothing():
    x, u, _ = rows_of(8, 64, 51865, dtype=torch.float16)
    x, u = x.to(DEV), u.to(DEV)
    want = ops.sample_rows(x, u, 0.9, 0, 0.95)
    out, logs = torch.zeros(64, dtype=torch.long, device=DEV), torch.zeros(64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_rows(x, u, 0.9, 0, 0.95, out=out, logprobs=logs)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    back = torch.arange(63, -1, -1, device=DEV)
    assert torch.equal(ops.sample_rows(x[back], u[back], 0.9, 0, 0.95), want[back])


def test_frequencies_follow_the_weights():
    """Evenly spaced numbers: each column is drawn for its share of them, to within one."""
    x = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5])
    n = 4000
    got = ops.sample_rows(x.to(DEV).expand(n, 5).contiguous(), ((torch.arange(n) + 0.5) / n).to(DEV), 0.7)
    share = torch.softmax(x.double() / 0.7, 0)
    drawn = torch.bincount(got.cpu(), minlength=5).double()
    assert ((drawn - share * n).abs() <= 1.0).all()
