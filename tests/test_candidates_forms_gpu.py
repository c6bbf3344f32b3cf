"""Forms of the candidates' attention that serve by themselves: own tokens without any prefix, and one query a request, over
types, head layouts and lengths.  Bounds as in test_candidates_gpu.py."""
import pytest
import torch

from int4_reference import cu
from speech_serving import ops
from test_candidates_gpu import DEV, Prefix, attend, near

pytestmark = pytest.mark.gpu
HEADS = [(2, 2, 64), (8, 1, 128), (9, 1, 64), (12, 4, 80), (40, 2, 32)]


@pytest.mark.parametrize("mine", [[1], [0, 1, 15, 16, 17, 130], [3000, 5, 511, 512, 513], [7] * 70])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_own_tokens_alone(mine, Hq, Hkv, D, dtype):
    c = Prefix(Hq + len(mine), [len(mine)], [0], mine, Hq, Hkv, D, dtype)
    q, k, v, _, _, _, table, lens = c.args()
    near(ops.shared_prefix_decode_attention(q, k, v, None, None, None, table, lens), c.want(first=len(mine)))


@pytest.mark.parametrize("B,T", [(1, 1500), (3, 1), (17, 129), (64, 333), (200, 40)])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_query_a_request(B, T, Hq, Hkv, D, dtype):
    g = torch.Generator().manual_seed(B + T + Hq)
    kv, q = torch.randn(B, 2, Hkv, T, D, generator=g).to(dtype), torch.randn(B, Hq, D, generator=g).to(dtype)
    lens = torch.randint(0, T + 1, (B,), generator=g)
    lens[0] = T
    d, valid = kv.to(DEV), lens.to(DEV, torch.int32)
    got = ops.cross_attention_packed(q.to(DEV), d[:, 0], d[:, 1], valid)
    assert torch.equal(got, ops.cross_attention_packed(q.to(DEV), d[:, 0], d[:, 1], valid, cu([1] * B).to(DEV)))
    near(got, [attend(q[b], *(kv[b, i, :, :n].transpose(0, 1) for i in (0, 1)), D ** -0.5) for b, n in enumerate(lens.tolist())])
