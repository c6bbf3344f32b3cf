"""paged_decode_attention_int4 with block ids out of range: the tokens of such a block take no part (nobody
else's cache is read in their place), the id is flagged, and the rest is as the 64-bit form has it."""
import pytest
import torch

from int4_reference import pack, unpack
from speech_serving import _native as N
from speech_serving import ops
from test_decode_int4_gpu import UNIT, make, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (12, 2)])
@pytest.mark.parametrize("D,bs", [(64, 8), (64, 16), (128, 16), (128, 32), (256, 8)])
@pytest.mark.parametrize("bad", [[0], [2], [-1], [1, 3, 4], list(range(8, 20)), [-2, -1]], ids=str)
def test_tokens_of_a_bad_block_take_no_part(Hq, Hkv, D, bs, bad):
    lens = [2500, 37 * bs - 3]  # the first is split over CTAs
    q, pool, tables = make(Hq + D + bs, lens, Hq, Hkv, D, bs, torch.float16)
    wild, kept, left = tables.clone(), [], []
    for b, n in enumerate(lens):
        blocks = -(-n // bs)
        gone = [c % blocks for c in bad]
        wild[b, gone] = torch.tensor([-1, pool.shape[0], 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32)[torch.arange(len(gone)) % 4]
        stay = [c for c in range(blocks) if c not in gone]
        row = torch.zeros(tables.shape[1], dtype=torch.int32)
        row[: len(stay)] = tables[b, stay]
        kept.append(row)
        left.append(sum(min(bs, n - c * bs) for c in stay))
    out, C, A, ds = reference(q, pool, torch.stack(kept), left, D, bs, D ** -0.5)
    # block 0 of the pool is in no table here; what it holds must not show
    stranger = int(next(i for i in range(pool.shape[0]) if not (tables == i).any()))
    order = torch.arange(pool.shape[0])
    order[[0, stranger]] = order[[stranger, 0]]
    swapped = wild.clone()
    swapped[wild == 0], swapped[wild == stranger] = stranger, 0
    kc, kp, vc, vp = unpack(pool[order], D, bs)
    kp[0], vp[0] = float("nan"), float("nan")
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.paged_decode_attention_int4(q.to(DEV), pack(kc, kp, vc, vp).to(DEV), swapped.to(DEV),
                                          torch.tensor(lens, dtype=torch.int32, device=DEV), error_word=word)
    assert ops.read_error_word(word) == N.SPD_DEVERR_BLOCK_ID
    u = 2.0 ** -22 if Hq // Hkv <= 4 else 2.0 ** -11
    bound = u * C + UNIT[torch.float16] * out.abs() * 1.001 + 2 * ds * A + 1e-6 * A
    assert ((got.cpu().double() - out).abs() <= bound).all()


def test_a_context_of_bad_blocks_alone_gives_zeros():
    lens = [50, 4000, 20]
    q, pool, tables = make(1, lens, 4, 2, 64, 16, torch.bfloat16)
    want = ops.paged_decode_attention_int4(q.to(DEV), pool.to(DEV), tables.to(DEV),
                                           torch.tensor(lens, dtype=torch.int32, device=DEV))
    tables[:2] = -9
    got = ops.paged_decode_attention_int4(q.to(DEV), pool.to(DEV), tables.to(DEV),
                                          torch.tensor(lens, dtype=torch.int32, device=DEV))
    assert not got[:2].any() and torch.equal(got[2], want[2])
