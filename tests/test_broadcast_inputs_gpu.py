"""Keys, values and queries that are broadcast views: strides of zero over heads or tokens."""
import pytest
import torch

import int4_reference as R
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [40, 64, 128])
def test_prompt_attention(D):
    lens = [70, 300, 1]
    n, cu = sum(lens), R.cu(lens).to(DEV)
    q, k, v = (torch.randn(n, h, D, device=DEV).half() for h in (4, 1, 1))
    for views in ((q, k.expand(n, 4, D), v.expand(n, 4, D)), (q, k[:1].expand(n, 1, D), v), (q[:, :1].expand(n, 4, D), k, v),
                  (q, k, v[:1, :1].expand(n, 2, D)[:, :1])):
        got = ops.prompt_attention(*views, cu)
        assert torch.equal(got, ops.prompt_attention(*(t.contiguous() for t in views), cu))


@pytest.mark.parametrize("bits", [4, 16])
def test_rotary_append(bits):
    cos, sin = (t.to(DEV) for t in R.angles(32, 64))
    q, k, v = (torch.randn(5, h, 64, device=DEV).half() for h in (4, 1, 1))
    table, first, cu = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), R.cu([5]).to(DEV)
    views = (q[:, :1].expand(5, 4, 64), k.expand(5, 2, 64), v[:1].expand(5, 1, 64).expand(5, 2, 64))
    found = []
    for q, k, v in (views, tuple(t.contiguous() for t in views)):
        if bits == 4:
            pool = ops.kv_pool_int4(1, 2, 64, 16)
            found.append((ops.rope_kv_append_int4(q, k, v, cos, sin, pool, table, first, cu), pool))
        else:
            pools = [torch.zeros(1, 16, 2, 64, dtype=torch.float16, device=DEV) for _ in range(2)]
            found.append((ops.rope_kv_append(q, k, v, cos, sin, *pools, table, first, cu), *pools))
    assert all(torch.equal(a, b) for a, b in zip(*found))
