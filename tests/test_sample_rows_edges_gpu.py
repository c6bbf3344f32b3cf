"""sample_rows at the ends of what it takes: random numbers, temperatures, widths, refusals, streams."""
import math

import pytest
import torch

from speech_serving import ops
from test_sample_rows_gpu import DEV, check, pick, rows_of

pytestmark = pytest.mark.gpu


def test_random_numbers_outside_their_range():
    x, _, _ = rows_of(0, 6, 4000, peaks=False)
    u = torch.tensor([math.nan, -1.0, -math.inf, 1.0, 7.0, math.inf])
    got = ops.sample_rows(x.to(DEV), u.to(DEV), 1.0, 50, 0.9).tolist()
    ends = [pick(x[r], 0.0 if r < 3 else 1.0 - 2.0 ** -24, 1.0, 50, 0.9) for r in range(6)]
    assert got == ends


@pytest.mark.parametrize("t", [1e-45, 1e-39, 1e-31, 1e-20])
def test_tiny_temperatures_leave_the_largest_values(t):
    x, _, _ = rows_of(1, 4, 900)
    x[:, 700] = x[:, 20] = x.max() + 1
    for k, p in ((0, 1.0), (5, 1.0), (0, 0.9), (2, 0.8)):
        for u, want in ((0.25, 20), (0.75, 700)):
            assert (ops.sample_rows(x.to(DEV), torch.full((4,), u, device=DEV), t, k, p) == want).all()


def test_an_infinite_temperature_makes_all_weights_equal():
    x, _, _ = rows_of(2, 8, 1000, peaks=False)
    u = (torch.arange(8) + 0.5) / 8
    assert ops.sample_rows(x.to(DEV), u.to(DEV), math.inf).tolist() == (u * 1000).floor().long().tolist()
    left = torch.argsort(-x, dim=1, stable=True)[:, :10].sort(1).values
    assert ops.sample_rows(x.to(DEV), u.to(DEV), math.inf, 10).tolist() == [int(left[r, int(u[r] * 10)]) for r in range(8)]


@pytest.mark.parametrize("dtype,cols", [(torch.float32, 440_000), (torch.bfloat16, 1 << 19), (torch.float16, 300_001)])
def test_widest_rows(dtype, cols):
    x, u, _ = rows_of(3, 2, cols, dtype=dtype)
    check(x, u, torch.tensor([1.0, 0.7]), torch.tensor([0, 1000]), torch.tensor([0.99, 0.9]))
    flat = torch.zeros(2, cols, dtype=dtype)
    check(flat, u, 1.0, 0, 0.9)


def test_one_column_and_no_rows():
    check(torch.tensor([[3.0], [-math.inf], [math.inf]]), torch.tensor([0.1, 0.5, 0.9]), 1.0, 3, 0.5, 0.1)
    assert ops.sample_rows(torch.zeros(0, 5, device=DEV), torch.zeros(0, device=DEV)).shape == (0,)


def test_outputs_where_they_are_asked_for():
    x, u, _ = rows_of(4, 9, 500)
    out, logs = torch.full((11,), -7, device=DEV), torch.full((11,), 7.0, device=DEV)
    got = ops.sample_rows(x.to(DEV), u.to(DEV), out=out[1:10], logprobs=logs[1:10])
    assert got.data_ptr() == out[1:].data_ptr() and (out[[0, 10]] == -7).all() and (logs[[0, 10]] == 7).all()
    assert out[1:10].tolist() == [pick(x[r], u[r]) for r in range(9)]


def test_streams_do_not_meet():
    cases = [rows_of(s, 40, 30000, dtype=torch.float16)[:2] for s in range(3)]
    cases = [(x.to(DEV), u.to(DEV)) for x, u in cases]
    want = [ops.sample_rows(x, u, 0.8, 0, 0.95) for x, u in cases]
    torch.cuda.synchronize()
    streams, found = [torch.cuda.Stream() for _ in cases], [[] for _ in cases]
    for _ in range(10):
        for s, (x, u), f in zip(streams, cases, found):
            with torch.cuda.stream(s):
                f.append(ops.sample_rows(x, u, 0.8, 0, 0.95))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for w, f in zip(want, found) for y in f)


def test_refusals():
    x, u = torch.zeros(4, 50, device=DEV), torch.zeros(4, device=DEV)
    longs, mask = torch.zeros(4, dtype=torch.long, device=DEV), torch.zeros(50, dtype=torch.bool, device=DEV)
    for args, kw in (
        ((x[0], u), {}), ((x[:, ::2], u), {}), ((x.long(), u), {}), ((x.double(), u), {}), ((x[:1].expand(4, 50), u), {}),
        ((x, u[:3]), {}), ((x, u.double()), {}), ((x, x[:, 0]), {}), ((x, u.cpu()), {}), ((x, u, u[:2]), {}), ((x, u, u.half()), {}),
        ((x, u, 1.0, u), {}), ((x, u, 1.0, 1.5), {}), ((x, u, 1.0, 2 ** 40), {}), ((x, u, 1.0, float("nan")), {}), ((x, u, "a"), {}),
        ((x, u, None), {}), ((x, u, 1.0, longs), {}), ((x, u, 1.0, 0, x[0]), {}), ((x, u, 1.0, 0, 1.0, longs), {}),
        ((x, u), dict(cols=0)), ((x, u), dict(cols=51)), ((x, u), dict(cols="3")), ((x[:, :0], u), {}), ((x, u), dict(skip=mask[:49])),
        ((x, u), dict(skip=mask.to(torch.uint8))), ((x, u), dict(skip=mask.cpu())), ((x, u), dict(out=longs[:3])),
        ((x, u), dict(out=longs.int())), ((x, u), dict(logprobs=u.half())), ((x, u), dict(logprobs=torch.zeros(5, device=DEV))),
        ((x, u), dict(logprobs=u)), ((x, u), dict(logprobs=x.view(-1)[:4])), ((x, u), dict(out=x.view(torch.long).view(-1)[:4])),
        ((x, u), dict(out=longs, logprobs=longs.view(torch.float32)[:4])), ((x, u, u), dict(logprobs=u)),
    ):
        with pytest.raises(RuntimeError):
            ops.sample_rows(*args, **kw)
    wide = torch.zeros(1, 1 << 19, device=DEV)
    with pytest.raises(RuntimeError, match="at most"):
        ops.sample_rows(wide, u[:1])
    with pytest.raises(RuntimeError, match="at most"):
        ops.sample_rows(torch.zeros(1, (1 << 19) + 8, device=DEV).half(), u[:1])
    torch.cuda.synchronize()


def test_columns_that_weigh_next_to_nothing_are_not_drawn():
    """Not even by a random number of zero: weights are in units of 2^-44 of the largest."""
    x = torch.full((3, 600), -100.0)
    x[0, 300], x[1, 599], x[2, 1] = 0.0, 0.0, 0.0
    x[2, 0] = -28.0  # 6.9e-13 of it: 12 units
    u = torch.tensor([0.0, 0.0, 0.0], device=DEV)
    for k, p in ((0, 1.0), (512, 1.0), (513, 1.0), (0, 0.99)):
        want = [300, 599, 0 if p == 1.0 else 1]
        assert ops.sample_rows(x.to(DEV), u, 1.0, k, p).tolist() == want
