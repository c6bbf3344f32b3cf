"""Rows of prompt_attention's output that belong to no sequence, and rows that see no key."""
import pytest
import torch

from speech_serving import ops

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
