"""shared_prefix_decode_attention over values that are infinite: a sum of weights times values with one infinity is that
infinity, with both signs NaN, and no other output changes a bit."""
import math

import pytest
import torch

from speech_serving import ops
from test_candidates_gpu import Prefix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (8, 1, 128), (6, 2, 40), (16, 1, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mine,prefix", [([20, 3], 0), ([1, 9], 30), ([1500, 600], 300)])
def test_infinite_values(Hq, Hkv, D, dtype, mine, prefix):
    # (scores of a few hundredths: with 1,800 keys each weighs some 2^-11 of the whole, none rounds to zero)
    c = Prefix(Hq, [2], [prefix], mine, Hq, Hkv, D, dtype, spread=0.02)
    a = c.args()
    if prefix == 0:
        a[3] = a[4] = a[5] = None
    want = ops.shared_prefix_decode_attention(*a)
    v = a[2].flatten(0, 1)
    own = [c.rows(c.tab[b], n) for b, n in enumerate(mine)]
    Gq = Hq // Hkv

    def expect(places, values):
        """`places`: (row of the pool, key/value head, dimension, sequences that see it, value)"""
        for row, h, d, seen, x in places:
            v[row, h, d] = x
            for b in seen:
                values[b, h * Gq : (h + 1) * Gq, d] += x
        got = ops.shared_prefix_decode_attention(*a)
        assert torch.equal(got.isnan(), values.isnan()) and torch.equal(got.nan_to_num(nan=7.0), values.nan_to_num(nan=7.0))

    h = Hkv - 1
    places = [(own[0][0], 0, 0, [0], math.inf), (own[1][-1], h, D - 1, [1], -math.inf), (own[1][1], h, 5, [1], math.inf),
              (own[1][2], h, 5, [1], -math.inf)]
    if prefix:
        shared = c.rows(c.ptab[0], prefix)
        places += [(shared[-1], h, 17, [0, 1], math.inf), (shared[3], 0, 18, [0, 1], -math.inf), (own[0][0], 0, 18, [0], -math.inf)]
    expect(places, want.float().clone().to(dtype))
