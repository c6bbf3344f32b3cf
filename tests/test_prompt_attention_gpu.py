"""prompt_attention against a plain 64-bit CPU form of the same packed prompts.

Tolerance per output (u the input type's unit: 2^-8 for bf16, 2^-11 for fp16):
  |off| <= u * A + u * |out| + 2 ds * A + n 2^-25 V
with A = sum p |v| (the weights p are rounded once to the input type), ds the error of a score
(2^-21 of scale * sum |q k|, for the fp32 sum of up to 128 products), and the last term the
weights that fp16 holds as subnormals (n keys, V the largest |v|; the largest weight is >= 1)."""
import math

import pytest
import torch

from int4_reference import cu
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(q, k, v, lens_q, lens_k, causal, scale):
    out, A, slack = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(3))
    G = q.shape[1] // k.shape[1]
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        if n and m:
            x, y, z = (t.double() for t in (q[a : a + n], k[b : b + m], v[b : b + m]))
            y, z = y.repeat_interleave(G, 1), z.repeat_interleave(G, 1)
            s = torch.einsum("ihd,jhd->hij", x, y) * scale
            size = torch.einsum("ihd,jhd->hij", x.abs(), y.abs()) * scale
            if causal:
                hidden = torch.ones(n, m, dtype=torch.bool).triu(m - n + 1)
                s.masked_fill_(hidden, -math.inf)
                size.masked_fill_(hidden, 0.0)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            out[a : a + n] = torch.einsum("hij,jhd->ihd", p, z)
            A[a : a + n] = torch.einsum("hij,jhd->ihd", p, z.abs())
            ds = 2.0 ** -21 * size.amax(-1).T[:, :, None]
            slack[a : a + n] = 2 * ds * A[a : a + n] + m * 2.0 ** -25 * z.abs().max() * (p.sum(-1).T[:, :, None] > 0)
        a, b = a + n, b + m
    return out, A, slack


def check(q, k, v, lens_q, lens_k=None, causal=True, scale=None, dev=None):
    lens_k = lens_q if lens_k is None else lens_k
    dq, dk, dv = dev if dev is not None else (t.to(DEV) for t in (q, k, v))
    got = ops.prompt_attention(dq, dk, dv, cu(lens_q).to(DEV), cu(lens_k).to(DEV), causal=causal, scale=scale)
    n = sum(lens_q)
    out, A, slack = reference(q, k, v, lens_q, lens_k, causal, scale or 1 / math.sqrt(q.shape[2]))
    u = UNIT[q.dtype]
    bound = u * A + u * out.abs() * 1.001 + slack
    off = (got.cpu().double() - out)[:n].abs()
    worst = (off / bound[:n].clamp(min=1e-300)).max() if n else 0
    assert (off <= bound[:n]).all(), worst
    return got


def make(seed, nq, nk, Hq, Hkv, D, dtype, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(nq, Hq, D, generator=g) * spread).to(dtype), torch.randn(nk, Hkv, D, generator=g).to(dtype),
            torch.randn(nk, Hkv, D, generator=g).to(dtype))


LENS = [[1], [4, 1, 0, 130], [128], [129, 127], [256, 257], [300, 5, 64, 511, 33]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (4, 1, 128), (6, 2, 64), (8, 1, 64), (3, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_matches_64_bits(lens, Hq, Hkv, D, causal, dtype):
    q, k, v = make(sum(lens) + Hq, sum(lens), sum(lens), Hq, Hkv, D, dtype)
    check(q, k, v, lens, causal=causal)


@pytest.mark.parametrize("D", [8, 16, 32, 40, 80, 96, 120])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_other_head_sizes(D, dtype):
    lens = [70, 200]
    q, k, v = make(D, 270, 270, 4, 2, D, dtype)
    check(q, k, v, lens)
    check(q, k, v, lens, causal=False)


@pytest.mark.parametrize("lens_q,lens_k", [([1, 1, 1], [1, 500, 128]), ([100, 3, 40], [1100, 130, 40]), ([257], [700]),
                                           ([200, 130, 5], [60, 0, 3]), ([300], [1])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 1, 128)])
def test_cached_prefixes_and_empty_rows(lens_q, lens_k, causal, Hq, Hkv, D):
    """More keys than queries (a prefix), and fewer: causal rows that see no key are zeros."""
    q, k, v = make(sum(lens_k), sum(lens_q), sum(lens_k), Hq, Hkv, D, torch.bfloat16)
    got = check(q, k, v, lens_q, lens_k, causal)
    a = 0
    for n, m in zip(lens_q, lens_k):
        empty = n if m == 0 else max(0, n - m) if causal else 0
        assert not got[a : a + empty].any()
        a += n


def test_longer_prompts_and_many_tiles():
    lens = [1500, 1, 2047, 640]
    n = sum(lens)
    q, k, v = make(1, n, n, 8, 2, 128, torch.bfloat16)
    check(q, k, v, lens)
    q, k, v = make(2, 1500, 1500, 12, 12, 64, torch.float16)
    check(q, k, v, [1500], causal=False)


def test_many_short_sequences():
    lens = [int(x) for x in torch.randint(0, 9, (150,), generator=torch.Generator().manual_seed(3))]
    n = sum(lens)
    q, k, v = make(3, n, n, 4, 4, 64, torch.float16)
    check(q, k, v, lens)


def test_peaked_flat_and_rising_scores():
    lens = [700]
    for spread in (1e-3, 12.0):
        q, k, v = make(4, 700, 700, 2, 1, 128, torch.bfloat16, spread)
        check(q, k, v, lens)
    q, k, v = make(5, 700, 700, 2, 2, 64, torch.float16)
    q, k = q.abs(), (k.abs() * torch.linspace(0, 4, 700)[:, None, None].half())  # the maximum rises at every step
    check(q, k, v, lens)
    check(q, -k, v, lens, causal=False, scale=0.5)


def test_strided_views():
    """q, k and v as views of one packed projection, head-major storage, and a sliced buffer."""
    lens = [90, 200, 3]
    n = sum(lens)
    qkv = torch.randn(n, 12, 64, generator=torch.Generator().manual_seed(6)).half()
    d = qkv.to(DEV)
    parts = (slice(0, 8), slice(8, 10), slice(10, 12))
    want = check(*(qkv[:, s] for s in parts), lens, dev=[d[:, s] for s in parts])
    major = [d[:, s].transpose(0, 1).contiguous().transpose(0, 1) for s in parts]
    wide = [torch.nn.functional.pad(d[:, s], (8, 24))[:, :, 8:72] for s in parts]
    for dev in (major, wide):
        assert torch.equal(want, ops.prompt_attention(*dev, cu(lens).to(DEV)))


def test_other_sequences_never_leak():
    """NaN and infinities in the keys, values and queries of the neighbouring sequences."""
    lens = [50, 77, 130]
    n = sum(lens)
    q, k, v = make(7, n, n, 4, 2, 64, torch.float16)
    want = check(q, k, v, lens)
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        t[:50] = bad
        t[127:] = bad
    got = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu(lens).to(DEV))
    assert torch.equal(got[50:127], want[50:127]) and torch.isnan(got[:50]).all()


@pytest.mark.parametrize("at", [0, 3, 5, 64, 130, 255])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_a_bad_key_shows_in_the_rows_that_see_it(at, bad, causal, D):
    """One NaN or infinite key element: rows that see the key give NaN, the others their result."""
    q, k, v = make(at, 256, 256, 2, 1, D, torch.bfloat16)
    q[:, :, 7] = q[:, :, 7].abs() + 0.1  # the infinite score is +inf
    out, A, slack = reference(q, k, v, [256], [256], causal, 1 / math.sqrt(D))
    bound = UNIT[q.dtype] * (A + out.abs() * 1.001) + slack
    k[at, 0, 7] = bad
    got = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu([256]).to(DEV), causal=causal)
    first = at if causal else 0
    assert torch.isnan(got[first:]).all()
    assert ((got.cpu().double() - out).abs() <= bound)[:first].all()


def test_scores_of_minus_infinity():
    """Keys whose scores are -inf have no weight; a row that has no other key gives zeros."""
    q, k, v = make(5, 200, 200, 2, 1, 64, torch.float16)
    q[:, :, 7] = q[:, :, 7].abs() + 0.1
    k[:150, 0, 7] = -math.inf
    got = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu([200]).to(DEV))
    assert not got[:150].any()
    keys = k[150:].clone()
    want = ops.prompt_attention(q[150:].contiguous().to(DEV), keys.to(DEV), v[150:].contiguous().to(DEV), cu([50]).to(DEV))
    # two ways to the same sums: the unit of the output and of a weight, twice each
    bound = 4 * UNIT[torch.float16] * v[150:].abs().max().item()
    assert (got[150:].float() - want.float()).abs().max().item() <= bound


def test_rows_of_no_sequence_are_left_alone():
    q, k, v = (t.to(DEV) for t in make(8, 100, 100, 2, 2, 64, torch.float16))
    out = torch.full_like(q, 7.0)
    ops.prompt_attention(q, k, v, torch.tensor([10, 60, 90], dtype=torch.int32, device=DEV), out=out)
    assert (out[:10] == 7).all() and (out[90:] == 7).all()
    want = ops.prompt_attention(q[10:90].contiguous(), k[10:90].contiguous(), v[10:90].contiguous(), cu([50, 30]).to(DEV))
    assert torch.equal(out[10:90], want)


def test_on_another_stream_and_in_a_graph():
    lens = [200, 40]
    q, k, v = make(9, 240, 240, 4, 1, 128, torch.bfloat16)
    want = check(q, k, v, lens)
    d, c = [t.to(DEV) for t in (q, k, v)], cu(lens).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.prompt_attention(*d, c)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(d[0])
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(*d, c, out=out, error_word=err)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and ops.read_error_word(err) == 0
    c.copy_(cu([100, 140]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.prompt_attention(*d, c))


def test_refusals():
    q, k, v = (t.to(DEV) for t in make(10, 20, 20, 4, 2, 64, torch.float16))
    c = cu([20]).to(DEV)
    ops.prompt_attention(q, k, v, c)
    for args, match in (((q.float(), k.float(), v.float(), c), "F16/BF16"), ((q, k[:, :, :32], v[:, :, :32], c), "expected"),
                        ((q[:, :3], k, v, c), "divide"), ((q, k, v.bfloat16(), c), "share a dtype"),
                        ((q, k, v, c.long()), "cu_seqlens_q"), ((q, k, v, c, cu([20, 0]).to(DEV)), "cu_seqlens_k"),
                        ((q.cpu(), k, v, c), "CUDA tensors"), ((q[..., :60], k[..., :60], v[..., :60], c), "not supported")):
        with pytest.raises(RuntimeError, match=match):
            ops.prompt_attention(*args)
    with pytest.raises(RuntimeError, match="scale"):
        ops.prompt_attention(q, k, v, c, scale=-1.0)
    with pytest.raises(RuntimeError, match="out must be"):
        ops.prompt_attention(q, k, v, c, out=torch.empty(20, 4, 64, device=DEV))
    with pytest.raises(RuntimeError, match="not supported"):
        wide = torch.zeros(4, 2, 136, device=DEV).half()
        ops.prompt_attention(wide, wide, wide, cu([4]).to(DEV))
    assert ops.prompt_attention(q[:0], k[:0], v[:0], cu([0]).to(DEV)).shape == (0, 4, 64)
    assert not ops.prompt_attention(q, k[:0], v[:0], c, cu([0]).to(DEV)).any()


@pytest.mark.parametrize("D", [64, 128])
def test_neighbours_change_no_rounding(D):
    """A sequence's rows are the same bits whatever the rows after it in its last tile hold."""
    lens = [400, 200]
    q, k, v = make(11, 600, 600, 4, 2, D, torch.bfloat16)
    args = [k.to(DEV), v.to(DEV), cu(lens).to(DEV)]
    want = ops.prompt_attention(q.to(DEV), *args)
    for other in (100.0, float("nan"), float("inf")):
        q[400:] = other
        assert torch.equal(ops.prompt_attention(q.to(DEV), *args)[:400], want[:400])
