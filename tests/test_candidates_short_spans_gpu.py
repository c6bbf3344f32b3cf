"""Spans of one step of keys between spans of many, several items a CTA, with one tile of rows or two: what the warps of the
spans' kernel hand over to one another from item to item.  Bounds as in test_candidates_gpu.py; every repeat has to give
the same bits and leave the error word at zero."""
import pytest
import torch

from int4_reference import cu
from speech_serving import _native as N
from speech_serving import ops
from test_candidates_gpu import DEV, EXPONENTIAL, UNIT

pytestmark = pytest.mark.gpu


def spans(seed, kind, dtype, D, requests, T=1500, Hkv=2):
    """Requests whose lengths mix 1 to 128 (one step) with 129 to T; `kind`: queries for one tile of 128 rows, for two, or both."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.where(torch.rand(requests, generator=g) < 0.7, torch.randint(1, 129, (requests,), generator=g),
                       torch.randint(129, T + 1, (requests,), generator=g))
    few, many = torch.randint(1, 41, (requests,), generator=g), torch.randint(129, 257, (requests,), generator=g)
    n = {"one tile": few, "two tiles": many, "both": torch.where(torch.rand(requests, generator=g) < 0.5, few, many)}[kind]
    on_device = torch.Generator(device=DEV).manual_seed(seed)
    kv = torch.randn(8, 2, Hkv, T, D, generator=on_device, device=DEV).to(dtype)
    q = torch.randn(int(n.sum()), Hkv, D, generator=on_device, device=DEV).to(dtype)
    slots = torch.randint(0, 8, (requests,), generator=g)
    return q, kv, lens, n, slots


def check(got, q, keys, n):
    """`keys(r)`: k and v [Hkv, T, D] of request r."""
    at, u, e = 0, UNIT[q.dtype], EXPONENTIAL[q.dtype]
    for r, rows in enumerate(n.tolist()):
        x, (y, z) = q[at : at + rows].double().transpose(0, 1), (t.double() for t in keys(r))
        scale = x.shape[2] ** -0.5
        p = torch.softmax(x @ y.mT * scale, -1)
        out, A = p @ z, p @ z.abs()
        ds = 2.0 ** -21 * (x.abs() @ y.abs().mT * scale).amax(-1, keepdim=True)
        bound = (u + 2 * e) * A + u * out.abs() * 1.001 + 2 * ds * A + y.shape[1] * 2.0 ** -25 * z.abs().max()
        off = (got[at : at + rows].double().transpose(0, 1) - out).abs()
        assert (off <= bound).all(), (r, (off / bound).max())
        at += rows


@pytest.mark.parametrize("kind", ["one tile", "two tiles", "both"])
@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 40)])
def test_cross_of_short_and_long_spans(kind, dtype, D):
    q, kv, lens, n, slots = spans(D, kind, dtype, D, 600)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = (q, kv[:, 0], kv[:, 1], lens.to(DEV, torch.int32), cu(n.tolist()).to(DEV), slots.to(DEV, torch.int32))
    first = ops.cross_attention_packed(*args, error_word=word)
    check(first, q, lambda r: kv[slots[r], :, :, : lens[r]], n)
    for _ in range(40):
        assert torch.equal(ops.cross_attention_packed(*args, error_word=word), first)
    assert ops.read_error_word(word) == 0


@pytest.mark.parametrize("kind", ["one tile", "two tiles", "both"])
@pytest.mark.parametrize("dtype,D,bs", [(torch.float16, 64, 16), (torch.bfloat16, 128, 32)])
def test_prefixes_of_short_and_long_spans(kind, dtype, D, bs):
    q, kv, lens, n, _ = spans(D + 1, kind, dtype, D, 300, T=1024)
    pool = kv.transpose(0, 1).transpose(2, 3).reshape(2, 8 * 1024 // bs, bs, 2, D).contiguous()
    g = torch.Generator().manual_seed(7)
    table = torch.randint(0, pool.shape[1], (300, 1024 // bs), generator=g).to(DEV, torch.int32)
    lens = lens.clamp(max=1024)
    B, word = q.shape[0], torch.zeros(1, dtype=torch.int32, device=DEV)
    none = torch.zeros(B, 0, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    args = (q, pool[0], pool[1], table, lens.to(DEV, torch.int32), cu(n.tolist()).to(DEV), *none)
    first = ops.shared_prefix_decode_attention(*args, error_word=word)
    check(first, q, lambda r: pool[:, table[r].long()].flatten(1, 2)[:, : lens[r]].transpose(1, 2), n)
    for _ in range(40):
        assert torch.equal(ops.shared_prefix_decode_attention(*args, error_word=word), first)
    assert ops.read_error_word(word) == 0


@pytest.mark.parametrize("kind", ["one tile", "two tiles", "both"])
@pytest.mark.parametrize("dtype,D,bs", [(torch.float16, 64, 8), (torch.bfloat16, 128, 32)])
def test_missing_pages_of_many_spans(kind, dtype, D, bs):
    """Block ids out of range in spans of odd and even numbers of steps, beside spans without any: each step leaves out its own
    pages and no other's."""
    requests, T = 120, 3200
    q, kv, lens, n, _ = spans(D + 2, kind, dtype, D, requests, T=T)
    g = torch.Generator().manual_seed(8)
    blocks = 8 * T // bs
    pool = kv.transpose(0, 1).transpose(2, 3).reshape(2, blocks, bs, 2, D).contiguous()
    table = torch.randint(0, blocks, (requests, T // bs), generator=g)
    gone = (torch.rand(requests, T // bs, generator=g) < 0.3) & (torch.arange(requests) % 2 == 0)[:, None]
    gone[:, 0] = False
    wild = torch.where(torch.rand(table.shape, generator=g) < 0.5, torch.tensor(-1), torch.tensor(blocks))
    B, word = q.shape[0], torch.zeros(1, dtype=torch.int32, device=DEV)
    none = torch.zeros(B, 0, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    args = (q, pool[0], pool[1], torch.where(gone, wild, table).to(DEV, torch.int32), lens.to(DEV, torch.int32),
            cu(n.tolist()).to(DEV), *none)

    def keys(r):
        left = (~gone[r]).repeat_interleave(bs)[: lens[r]].to(DEV)
        return pool[:, table[r].to(DEV)].flatten(1, 2)[:, : lens[r]][:, left].transpose(1, 2)

    first = ops.shared_prefix_decode_attention(*args, error_word=word)
    check(first, q, keys, n)
    for _ in range(40):
        assert torch.equal(ops.shared_prefix_decode_attention(*args, error_word=word), first)
    assert ops.read_error_word(word) == N.SPD_DEVERR_BLOCK_ID
