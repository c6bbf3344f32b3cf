"""4-bit decode attention over the longest context that the tables can say: 2^31 - 32 tokens.

The table repeats 64 blocks, so the result is the attention over those.  It is a ratio of two fp32 sums
over the context's 2^19 chunks: each may be off by 2^19 units of 2^-24, and the ratio by twice that."""
import pytest
import torch

import int4_reference as R
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_the_longest_context():
    bs, D, columns = 32, 64, (2 ** 31 - 1) // 32
    pool, k, v = R.random_pool(torch.Generator().manual_seed(0), 64, bs, 1, D)
    v = v + 3.0
    pool = R.pack(*R.quantise(k.float()), *R.quantise(v.float()))
    _, _, vc, vp = R.unpack(pool, D, bs)
    v = R.values(vc, vp).flatten(0, 2)
    kc, kp, _, _ = R.unpack(pool, D, bs)
    k = R.values(kc, kp).flatten(0, 2)
    q = torch.randn(1, 1, D, generator=torch.Generator().manual_seed(1)).half()
    want = torch.softmax(k @ q[0, 0].double() / 8, 0) @ v
    table = (torch.arange(columns, dtype=torch.int32, device=DEV) % 64)[None]
    lens = torch.tensor([columns * bs], dtype=torch.int32, device=DEV)
    out = torch.zeros(1, 1, D, dtype=torch.float16, device=DEV)
    ops.paged_decode_attention_int4(q.to(DEV), pool.to(DEV), table, lens, out=out)
    assert ((out[0, 0].cpu().double() - want).abs() <= 2 * 2.0 ** -5 * want.abs()).all()
