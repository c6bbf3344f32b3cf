"""Calls of the rotary append and the 4-bit gather without tokens, or without sequences, do nothing."""
import pytest
import torch

import int4_reference as R
from speech_serving import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("B,columns", [(0, 4), (0, 0), (3, 4), (3, 0)])
@pytest.mark.parametrize("packed", [True, False])
def test_append_without_tokens(bits, B, columns, packed):
    if B and not packed:
        pytest.skip("without cu_seqlens there is a token for every sequence")
    cos, sin = (t.to(DEV) for t in R.angles(8, 64))
    qkv = torch.randn(5, 4, 64, device=DEV).half()[:0]
    tables = torch.zeros(B, columns, dtype=torch.int32, device=DEV)
    positions = torch.zeros(B, dtype=torch.int32, device=DEV)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV) if packed else None
    for q in (qkv[:, :2], None):
        for tab in ((cos, sin), (cos[:0], sin[:0])):
            if bits == 4:
                pool = torch.full_like(ops.kv_pool_int4(3, 1, 64, 16), 5)
                out = ops.rope_kv_append_int4(q, qkv[:, 2:3], qkv[:, 3:], *tab, pool, tables, positions, cu)
                assert (pool == 5).all()
            else:
                pools = [torch.full((3, 16, 1, 64), 5.0, dtype=torch.float16, device=DEV) for _ in range(2)]
                out = ops.rope_kv_append(q, qkv[:, 2:3], qkv[:, 3:], *tab, *pools, tables, positions, cu)
                assert all((p == 5).all() for p in pools)
            assert (out is None) if q is None else out.shape == (0, 2, 64)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("columns", [0, 4])
def test_append_of_tokens_of_no_sequence(bits, columns):
    """A batch of no sequences: rows of q come back as zeros, nothing is written."""
    cos, sin = (t.to(DEV) for t in R.angles(8, 64))
    qkv = torch.randn(5, 4, 64, device=DEV).half()
    tables, positions, cu = torch.zeros(0, columns, dtype=torch.int32, device=DEV), ints(), ints(0)
    if bits == 4:
        pool = torch.full_like(ops.kv_pool_int4(3, 1, 64, 16), 5)
        out = ops.rope_kv_append_int4(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], cos, sin, pool, tables, positions, cu)
        assert (pool == 5).all()
    else:
        pools = [torch.full((3, 16, 1, 64), 5.0, dtype=torch.float16, device=DEV) for _ in range(2)]
        out = ops.rope_kv_append(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], cos, sin, *pools, tables, positions, cu)
        assert all((p == 5).all() for p in pools)
    assert out.shape == (5, 2, 64) and not out.any()


@pytest.mark.parametrize("B,columns", [(0, 4), (2, 4), (2, 0)])
def test_gather_without_tokens(B, columns):
    """A batch that has no cached prefix."""
    pool = ops.kv_pool_int4(3, 2, 128, 16)
    tables = torch.zeros(B, columns, dtype=torch.int32, device=DEV)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    for kw in ({}, dict(starts=torch.zeros(B, dtype=torch.int32, device=DEV)),
               dict(k_out=torch.empty(0, 2, 128, device=DEV), v_out=torch.empty(0, 2, 128, device=DEV))):
        k, v = ops.kv_gather_int4(pool, tables, cu, 0, 128, torch.float32, **kw)
        assert k.shape == v.shape == (0, 2, 128)
    if B == 0:  # rows of no sequence are left alone
        k, v = (torch.full((4, 2, 128), 7.0, device=DEV) for _ in range(2))
        ops.kv_gather_int4(pool, tables, cu, 4, 128, torch.float32, k_out=k, v_out=v)
        assert (k == 7).all() and (v == 7).all()


def test_missing_tables_are_still_refused():
    cos, sin = (t.to(DEV) for t in R.angles(8, 64))
    x = torch.randn(2, 1, 64, device=DEV).half()
    pool, none = ops.kv_pool_int4(3, 1, 64, 16), torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        ops.rope_kv_append_int4(None, x, x, cos, sin, pool, none, ints(0, 0))
    with pytest.raises(RuntimeError):
        ops.kv_gather_int4(pool, none, ints(0, 1, 2), 2, 64, torch.float16)
    with pytest.raises(RuntimeError):
        ops.rope_kv_append_int4(None, x, x, cos[:0], sin[:0], pool, torch.zeros(2, 1, dtype=torch.int32, device=DEV), ints(0, 0))
