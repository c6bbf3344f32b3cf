"""paged_decode_attention_int4 against a plain 64-bit CPU form over the same pool.

Tolerance per output, from the kernel's roundings (u the unit of the weights it multiplies:
2^-22 where a head takes two columns, 2^-11 otherwise; U the output type's unit):
  |off| <= u * C + U * |out| + 2 ds * A + 1e-6 * A
with C = sum p scale c and A = sum p (scale c + |zero|) of the softmax p, and ds the error of a
score: 2^-20 of scale_softmax * sum |q| (15 scale + |zero|), for the fp32 sums of 64 products
and of the two terms."""
import math

import pytest
import torch

import int4_reference as R
from speech_serving import _native as N
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(q, pool, tables, lens, D, bs, scale):
    """(out, C, A, ds) in 64 bits, [B, Hq, D]."""
    kc, kp, vc, vp = R.unpack(pool, D, bs)
    B, Hq, _ = q.shape
    Hkv = pool.shape[1]
    G = Hq // Hkv
    out, C, A, ds = (torch.zeros(B, Hq, D, dtype=torch.float64) for _ in range(4))
    k_all, v_all = R.values(kc, kp), R.values(vc, vp)
    vs = R.values(vc, torch.stack((vp[..., 0], torch.zeros_like(vp[..., 1])), -1))
    wide_k = R.values(torch.full_like(kc, 15), torch.stack((kp[..., 0], kp[..., 1].abs()), -1))
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        rows = tables[b].long()
        k, v, s, wk = (x[rows].flatten(0, 1)[:n].repeat_interleave(G, 1) for x in (k_all, v_all, vs, wide_k))
        x = q[b].double()
        p = torch.softmax(torch.einsum("hd,thd->ht", x, k) * scale, -1)
        out[b] = torch.einsum("ht,thd->hd", p, v)
        C[b] = torch.einsum("ht,thd->hd", p, s)
        A[b] = C[b] + torch.einsum("ht,thd->hd", p, (v - s).abs())
        ds[b] = (2.0 ** -20 * scale * torch.einsum("hd,thd->ht", x.abs(), wk).amax(-1))[:, None]
    return out, C, A, ds


def check(q, pool, tables, lens, bs, dtype, scale=None, **kw):
    D = q.shape[2]
    sm = scale or 1 / math.sqrt(D)
    got = ops.paged_decode_attention_int4(q.to(DEV), pool.to(DEV), tables.to(DEV),
                                          torch.tensor(lens, dtype=torch.int32, device=DEV), scale=scale, **kw)
    out, C, A, ds = reference(q, pool, tables, lens, D, bs, sm)
    G = q.shape[1] // pool.shape[1]
    u = 2.0 ** -22 if dtype == torch.float32 or G <= 4 else 2.0 ** -11
    bound = u * C + UNIT[dtype] * out.abs() * 1.001 + 2 * ds * A + 1e-6 * A
    off = (got.cpu().double() - out).abs()
    assert (off <= bound).all(), (off / bound.clamp(min=1e-300)).max()
    return got


def make(seed, lens, Hq, Hkv, D, bs, dtype, spread=1.0, qscale=1.0):
    g = torch.Generator().manual_seed(seed)
    tables, blocks = R.tables(g, lens, bs)
    pool, *_ = R.random_pool(g, blocks, bs, Hkv, D, spread)
    return (torch.randn(len(lens), Hq, D, generator=g) * qscale).to(dtype), pool, tables


HEADS = [(1, 1), (12, 12), (8, 2), (10, 5), (12, 2), (16, 2), (9, 1), (20, 1)]  # groups of 1, 4, 2, 6, 8, 9, 20


@pytest.mark.parametrize("Hq,Hkv", HEADS)
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (128, 8), (64, 32), (256, 16)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_matches_64_bits(Hq, Hkv, D, bs, dtype):
    lens = [1, 0, bs - 1, bs, bs + 1, 63, 64, 65, 257, 300]
    q, pool, tables = make(Hq * 100 + D + bs, lens, Hq, Hkv, D, bs, dtype)
    got = check(q, pool, tables, lens, bs, dtype)
    assert not got[1].any()


@pytest.mark.parametrize("lens", [[5000], [4097, 0, 1], [3000, 17, 2049, 256, 255, 512]])
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (16, 2)])
def test_chunks_of_long_contexts_are_joined(lens, Hq, Hkv):
    q, pool, tables = make(sum(lens), lens, Hq, Hkv, 128, 16, torch.bfloat16)
    a = check(q, pool, tables, lens, 16, torch.bfloat16)
    ws = ops.decode_int4_workspace(len(lens), Hq, Hkv, 128, 16, tables.shape[1], torch.bfloat16, torch.device(DEV))
    for _ in range(3):  # the arrival counters come back to zero, and the result does not change
        assert torch.equal(a, check(q, pool, tables, lens, 16, torch.bfloat16, workspace=ws))
    assert not ws[256 : 256 + 4 * len(lens) * Hq].any() and ops.read_error_word(ws) == 0


@pytest.mark.parametrize("spread,qscale", [(1e-3, 1.0), (100.0, 0.3), (1.0, 1e-4), (0.05, 3e4), (2.0, 8.0)])
@pytest.mark.parametrize("Hq", [4, 16])
def test_magnitudes(spread, qscale, Hq):
    """Values and queries far from 1: peaked and flat softmaxes, small and large scales."""
    lens = [200, 700]
    for dtype in (torch.bfloat16, torch.float32):
        q, pool, tables = make(3, lens, Hq, 2, 64, 16, dtype, spread, qscale)
        check(q, pool, tables, lens, 16, dtype)


def test_rising_scores_and_scales():
    """Scores and value scales that rise along the context, so that the running maximum and
    the weights' exponent are raised at every step."""
    g = torch.Generator().manual_seed(4)
    lens, bs, D = [1500], 16, 64
    tables, blocks = R.tables(g, lens, bs)
    order = torch.zeros(blocks, dtype=torch.double)
    order[tables[0].long()] = torch.arange(tables.shape[1], dtype=torch.double)
    ramp = (order / tables.shape[1])[:, None, None, None].float()
    made = R.quantise(torch.randn(blocks, bs, 1, D, generator=g) + 6 * ramp) + R.quantise(
        torch.randn(blocks, bs, 1, D, generator=g) * 2 ** (20 * ramp - 10))
    pool = R.pack(*made)
    for Hq in (2, 8):
        q = torch.ones(1, Hq, D).half() * torch.linspace(0.1, 2.0, Hq)[:, None].half()
        check(q, pool, tables, lens, bs, torch.float16)


def test_what_lies_past_the_context_never_counts():
    """Slots past the context hold NaN and infinite parameters; unused table entries are wild."""
    lens, bs, D, Hkv = [1, 20, 77, 130], 16, 128, 2
    q, pool, tables = make(5, lens, 8, Hkv, D, bs, torch.float16)
    want = check(q, pool, tables, lens, bs, torch.float16)
    kc, kp, vc, vp = R.unpack(pool, D, bs)
    seen = torch.zeros(pool.shape[0], bs, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            seen[tables[b, t // bs], t % bs] = True
    for x, bad in ((kp, float("nan")), (vp, float("inf"))):
        x[~seen] = bad
    vp[~seen, :, :, 1] = float("nan")
    wild = tables.clone()
    for b, n in enumerate(lens):
        wild[b, -(-n // bs):] = -12345
    got = ops.paged_decode_attention_int4(q.to(DEV), R.pack(kc, kp, vc, vp).to(DEV), wild.to(DEV),
                                          torch.tensor(lens, dtype=torch.int32, device=DEV))
    assert torch.equal(got, want)


def test_nan_stays_in_its_sequence_and_head():
    lens, bs, D = [40, 40], 16, 64
    q, pool, tables = make(6, lens, 4, 2, D, bs, torch.float16)
    kc, kp, vc, vp = R.unpack(pool, D, bs)
    vp[tables[0, 1], 3, 1, 0, 1] = float("nan")
    got = ops.paged_decode_attention_int4(q.to(DEV), R.pack(kc, kp, vc, vp).to(DEV), tables.to(DEV),
                                          torch.tensor(lens, dtype=torch.int32, device=DEV))
    assert torch.isnan(got[0, 2:]).all() and torch.isfinite(got[0, :2]).all() and torch.isfinite(got[1]).all()


def test_bad_block_and_length_are_flagged():
    lens, bs = [40, 10], 16
    q, pool, tables = make(7, lens, 2, 2, 64, bs, torch.float16)
    ws = ops.decode_int4_workspace(2, 2, 2, 64, bs, tables.shape[1], torch.float16, torch.device(DEV))
    bad = tables.clone()
    bad[0, 1] = 10_000
    run = lambda t, n: ops.paged_decode_attention_int4(  # noqa: E731
        q.to(DEV), pool.to(DEV), t.to(DEV), torch.tensor(n, dtype=torch.int32, device=DEV), workspace=ws)
    out = run(bad, lens)
    assert ops.read_error_word(ws) == N.SPD_DEVERR_BLOCK_ID and torch.equal(out[1], run(tables, lens)[1])
    ws.zero_()
    full = tables.shape[1] * bs
    long = run(tables, [full + 1, 10])
    assert ops.read_error_word(ws) == N.SPD_DEVERR_LENGTH and torch.equal(long, run(tables, [full, 10]))


def test_on_another_stream_and_in_a_graph():
    lens, bs = [300, 5, 64], 16
    q, pool, tables = make(8, lens, 8, 2, 128, bs, torch.bfloat16)
    want = check(q, pool, tables, lens, bs, torch.bfloat16)
    args = [q.to(DEV), pool.to(DEV), tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)]
    ws = ops.decode_int4_workspace(3, 8, 2, 128, bs, tables.shape[1], torch.bfloat16, torch.device(DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_decode_attention_int4(*args)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(args[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_decode_attention_int4(*args, out=out, workspace=ws)
    for n in (lens, [64, 64, 1]):
        args[3].copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.paged_decode_attention_int4(*args))


def test_refusals():
    lens = [40, 10]
    q, pool, tables = make(9, lens, 4, 2, 64, 16, torch.float16)
    good = dict(q=q.to(DEV), pool=pool.to(DEV), block_tables=tables.to(DEV),
                context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    ops.paged_decode_attention_int4(**good)
    three = torch.zeros(2, 3, 64, device=DEV).half()
    for change, match in ((dict(q=three), "divide"), (dict(q=good["q"][:, :, :32].contiguous()), "fit no block size"),
                          (dict(q=good["q"].transpose(0, 1)), "contiguous"), (dict(q=good["q"].double()), "not supported"),
                          (dict(context_lens=good["context_lens"].long()), "context_lens"),
                          (dict(block_tables=good["block_tables"].long()), "block_tables"),
                          (dict(out=torch.empty(2, 4, 64, device=DEV)), "out must be"), (dict(pool=pool), "CUDA tensors"),
                          (dict(workspace=torch.zeros(64, dtype=torch.uint8, device=DEV)), "workspace")):
        with pytest.raises(RuntimeError, match=match):
            ops.paged_decode_attention_int4(**{**good, **change})
    empty = ops.paged_decode_attention_int4(good["q"][:0], good["pool"], good["block_tables"][:0], good["context_lens"][:0])
    assert empty.shape == (0, 4, 64)
