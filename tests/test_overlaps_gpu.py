"""Outputs over inputs that other CTAs still read are refused; an output in place of the queries is not."""
import pytest
import torch

import int4_reference as R
from speech_serving import ops
from test_decode_int4_gpu import make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [40, 64, 128])
def test_prompt_attention(D):
    lens = [300, 1, 77, 700]
    n = sum(lens)
    buf = torch.randn(4, n, 4, D, device=DEV).half()
    q, k, v = buf[0], buf[1], buf[2]
    cu = R.cu(lens).to(DEV)
    want = ops.prompt_attention(q, k, v, cu)
    flat = buf.view(4 * n, 4, D)
    for out in (k, v, flat[n // 2 : n // 2 + n], flat[n - 1 : 2 * n - 1], flat[1 : n + 1]):
        with pytest.raises(RuntimeError, match="apart from k and v"):
            ops.prompt_attention(q, k, v, cu, out=out)
    assert torch.equal(ops.prompt_attention(q, k, v, cu, out=buf[3]), want)
    got = ops.prompt_attention(q, k, v, cu, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("Hq", [4, 12])
def test_paged_decode_attention_int4(Hq):
    lens = [3000, 40, 0]
    q, pool, tables = make(1, lens, Hq, 2, 64, 16, torch.float16)
    buf = torch.zeros(8, Hq, 64, dtype=torch.float16, device=DEV)
    buf[:3] = q.to(DEV)
    args = (pool.to(DEV), tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    want = ops.paged_decode_attention_int4(buf[:3], *args)
    with pytest.raises(RuntimeError, match="apart from q"):
        ops.paged_decode_attention_int4(buf[:3], *args, out=buf[1:4])
    assert torch.equal(ops.paged_decode_attention_int4(buf[:3], *args, out=buf[3:6]), want)
    assert torch.equal(ops.paged_decode_attention_int4(buf[:3], *args, out=buf[:3]), want)


@pytest.mark.parametrize("bits", [4, 16])
def test_rotary_append_and_gather(bits):
    cos, sin = (t.to(DEV) for t in R.angles(16, 64))
    buf = torch.randn(8, 5, 2, 64, device=DEV).half()
    q, k, v = buf[0], buf[1], buf[2]
    table, first, cu = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), R.cu([5]).to(DEV)
    pool = ops.kv_pool_int4(1, 2, 64, 16)
    pools = [torch.zeros(1, 16, 2, 64, dtype=torch.float16, device=DEV) for _ in range(2)]

    def append(out):
        if bits == 4:
            return ops.rope_kv_append_int4(q, k, v, cos, sin, pool, table, first, cu, q_out=out)
        return ops.rope_kv_append(q, k, v, cos, sin, *pools, table, first, cu, q_out=out)

    flat = buf.view(40, 2, 64)
    for out in (k, v, flat[3:8], flat[12:17]):
        with pytest.raises(RuntimeError, match="apart from q"):
            append(out)
    assert torch.equal(append(buf[3]), append(None))
    if bits == 4:
        with pytest.raises(RuntimeError, match="overlap"):
            ops.kv_gather_int4(pool, table, cu, 5, 64, torch.float16, k_out=flat[:5], v_out=flat[4:9])
        got = ops.kv_gather_int4(pool, table, cu, 5, 64, torch.float16, k_out=flat[:5], v_out=flat[5:10])
        assert all(torch.equal(a, b) for a, b in zip(got, ops.kv_gather_int4(pool, table, cu, 5, 64, torch.float16)))
