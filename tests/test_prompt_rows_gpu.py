"""Rows of prompt_attention's output that belong to no sequence, and rows that see no key."""
import pytest
import torch

from int4_reference import cu
from speech_serving import ops
from test_prompt_attention_gpu import UNIT, make, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("cu_q", [[10, 60, 90], [0, 0, 100], [0, 100, 100], [3, 3, 3], [0, 1, 2]], ids=str)
@pytest.mark.parametrize("heads,D", [(2, 64), (5, 24), (32, 128)])
def test_without_any_key_other_rows_are_left_alone(cu_q, heads, D):
    q = torch.randn(100, heads, D, device=DEV).half()
    k = torch.randn(4, heads, D, device=DEV).half()[:0]
    out = torch.full_like(q, 7.0)
    cq = torch.tensor(cu_q, dtype=torch.int32, device=DEV)
    for causal in (True, False):
        ops.prompt_attention(q, k, k, cq, torch.zeros(3, dtype=torch.int32, device=DEV), causal=causal, out=out)
        assert not out[cu_q[0] : cu_q[2]].any()
        assert (out[: cu_q[0]] == 7).all() and (out[cu_q[2] :] == 7).all()


def check_bad_values(lens_q, lens_k, Hq, Hkv, D, dtype, at, seed, causal=True, rows=None):
    """`at`: (key, head, dimension, value) of the packed v.  Dimensions of rows that do not see such a key
    hold the 64-bit form's result of the finite values; the others are what an infinity or a NaN makes."""
    q, k, v = make(seed, sum(lens_q), sum(lens_k), Hq, Hkv, D, dtype)
    bad = v.clone()
    for key, head, dim, value in at:
        v[key, head, dim] = 0
        bad[key, head, dim] = value
    got = ops.prompt_attention(q.to(DEV), k.to(DEV), bad.to(DEV), cu(lens_q).to(DEV), cu(lens_k).to(DEV), causal=causal).cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)  # sees a bad value
    nan, pos, neg = (torch.zeros(got.shape, dtype=torch.bool) for _ in range(3))
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        for key, head, dim, value in at:
            if b <= key < b + m:
                first = max(0, key - b - (m - n)) if causal else 0
                heads = slice(head * (Hq // Hkv), (head + 1) * (Hq // Hkv))
                hit[a + first : a + n, heads, dim] = True
                for mask, is_it in ((nan, value != value), (pos, value == float("inf")), (neg, value == -float("inf"))):
                    mask[a + first : a + n, heads, dim] |= is_it
        a, b = a + n, b + m
    assert not torch.isfinite(got[hit]).any()
    assert torch.isnan(got[nan | (pos & neg)]).all()
    assert (got[hit & pos & ~neg & ~nan] != -float("inf")).all() and (got[hit & neg & ~pos & ~nan] != float("inf")).all()
    if rows is not None:  # the 64-bit form of some sequences alone
        keep_q, keep_k = rows
        q, k, v, got, hit = q[keep_q[0] : keep_q[1]], k[keep_k[0] : keep_k[1]], v[keep_k[0] : keep_k[1]], got[keep_q[0] : keep_q[1]], hit[keep_q[0] : keep_q[1]]
        lens_q, lens_k = [keep_q[1] - keep_q[0]], [keep_k[1] - keep_k[0]]
    out, A, slack = reference(q, k, v, lens_q, lens_k, causal, D ** -0.5)
    bound = UNIT[dtype] * (A + out.abs() * 1.001) + slack
    assert ((got.double() - out).abs() <= bound)[~hit].all()
    return got


NAN, INF = float("nan"), float("inf")
PLACES = {  # sequences of 300 keys and up: the first, the last, around the borders of steps and tiles
    "one NaN": [(130, 0, 3, NAN)],
    "one infinity": [(255, 0, 0, -INF)],
    "last key": [(299, 0, 7, INF)],
    "first key": [(0, 0, 5, NAN)],
    "many": [(i, 0, i % 8, [NAN, INF, -INF][i % 3]) for i in range(40, 300, 7)],
    "both infinities in a dimension": [(64, 0, 2, INF), (200, 0, 2, -INF)],
}


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (4, 1, 128), (3, 1, 128), (8, 1, 64), (2, 1, 40), (2, 1, 96)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(place, Hq, Hkv, D, dtype):
    check_bad_values([300], [300], Hq, Hkv, D, dtype, PLACES[place], 1)
    check_bad_values([40, 300], [300, 300], Hq, Hkv, D, dtype, PLACES[place], 2)               # a prefix
    check_bad_values([450, 20], [300, 20], Hq, Hkv, D, dtype, PLACES[place], 3)                # rows that see no key
    check_bad_values([1, 513], [301, 700], Hq, Hkv, D, dtype, PLACES[place] + [(600, 0, 1, NAN)], 4)
    check_bad_values([300], [300], Hq, Hkv, D, dtype, PLACES[place], 5, causal=False)


@pytest.mark.parametrize("heads,D", [(16, 64), (16, 128), (12, 32)])
def test_and_where_a_cta_takes_several_items(heads, D):
    """More items than CTAs run at once, so that items of other lengths come before and after."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    lens = [700, 90, 513] + [300] * (3 * sms // heads + 1)
    at = [(i, i % heads, i % 8, [NAN, INF, -INF][i % 3]) for i in range(100, 1300, 11)]
    check_bad_values(lens, lens, heads, heads, D, torch.bfloat16, at, 6, rows=((0, 700), (0, 700)))
    check_bad_values(lens, lens, heads, heads, D, torch.float16, at, 7, rows=((790, 1303), (790, 1303)))
    got = check_bad_values(lens, lens, heads, heads, D, torch.float16, at, 8, rows=((1303, 1603), (1303, 1603)))
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("value", [NAN, INF], ids=str)
def test_nothing_but_bad_values_costs_no_multiple(value):
    """A batch whose v holds nothing finite (a model that has diverged): the repairs are a few milliseconds."""
    lens = [2000, 700, 3000]
    n = sum(lens)
    q, k, v = (t.to(DEV) for t in make(9, n, n, 16, 4, 128, torch.bfloat16))
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    bad = torch.full_like(v, value)
    c = cu(lens).to(DEV)
    ops.prompt_attention(q, k, bad, c)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got = ops.prompt_attention(q, k, bad, c, error_word=word)
    end.record()
    end.synchronize()
    assert ops.read_error_word(word) == 0 and not torch.isfinite(got).any()
    print(f"{start.elapsed_time(end):.2f} ms")
    assert start.elapsed_time(end) < 100
