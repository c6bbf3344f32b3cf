"""Host-side checks of the operators for several candidates of a request: they come before any CUDA call."""
import pytest
import torch

from speech_serving import _native as N
from speech_serving import ops

INVALID, UNSUPPORTED, F16, F32 = N.SPD_ERR_INVALID_ARG, N.SPD_ERR_UNSUPPORTED, N.SPD_F16, N.SPD_F32
P = 4096  # an address that is only looked at


def prefix(lib, *, q=P, qst=64, qsh=64, k=P, v=P, ptab=P, plens=P, cu=P, tab=P, lens=P, out=P, B=2, G=1, Hq=2, Hkv=1, D=64, bs=16,
           pcols=4, cols=4, blocks=8, scale=0.125, dtype=F16, ws=None, ws_bytes=0):
    return lib.spd_shared_prefix_attn(q, qst, qsh, k, v, ptab, plens, cu, tab, lens, out, B, G, Hq, Hkv, D, bs, pcols, cols, blocks,
                                      scale, dtype, ws, ws_bytes, None, None)


def cross(lib, *, q=P, qst=64, qsh=64, k=P, v=P, sb=640, sh=640, st=64, lens=P, cu=P, slots=None, out=P, n=4, B=2, S=2, T=10, Hq=1,
          Hkv=1, D=64, scale=0.125, dtype=F16, ws=None, ws_bytes=0):
    return lib.spd_cross_attn_packed(q, qst, qsh, k, v, sb, sh, st, lens, cu, slots, out, n, B, S, T, Hq, Hkv, D, scale, dtype, ws,
                                     ws_bytes, None, None)


def sample(lib, *, x=P, rows=2, cols=10, ld=10, skip=None, u=P, out=P, logprobs=None, dtype=F16):
    return lib.spd_sample_rows(x, rows, cols, ld, skip, u, None, 1.0, None, 0, None, 1.0, None, 0.0, out, logprobs, dtype, None)


@pytest.mark.parametrize("want,bad", [
    (UNSUPPORTED, dict(dtype=F32)), (UNSUPPORTED, dict(dtype=99)), (INVALID, dict(B=-1)), (INVALID, dict(G=-1)),
    (INVALID, dict(Hq=3, Hkv=2)), (INVALID, dict(Hkv=0)), (INVALID, dict(D=0)), (UNSUPPORTED, dict(D=136)), (UNSUPPORTED, dict(D=60)),
    (UNSUPPORTED, dict(bs=24)), (UNSUPPORTED, dict(bs=4)), (UNSUPPORTED, dict(bs=256)), (UNSUPPORTED, dict(Hq=129)),
    (UNSUPPORTED, dict(B=65537)), (UNSUPPORTED, dict(cols=1 << 28)), (UNSUPPORTED, dict(pcols=1 << 28)), (INVALID, dict(scale=0.0)),
    (INVALID, dict(scale=-1.0)), (INVALID, dict(scale=float("nan"))), (INVALID, dict(q=None)), (INVALID, dict(k=None)),
    (INVALID, dict(v=None)), (INVALID, dict(ptab=None)), (INVALID, dict(plens=None)), (INVALID, dict(cu=None)), (INVALID, dict(tab=None)),
    (INVALID, dict(lens=None)), (INVALID, dict(out=None)), (INVALID, dict(blocks=0)), (INVALID, dict(qst=63)), (INVALID, dict(qsh=-64)),
    (INVALID, dict(q=P + 2)), (INVALID, dict(k=P + 8)), (INVALID, dict(out=P + 4)), (INVALID, dict(ws=P + 1)),
    (UNSUPPORTED, dict(B=65536, G=1, Hq=4096, Hkv=4096, qst=4096 * 64, pcols=1 << 20)),
])
def test_prefix_refusals(want, bad):
    lib = N.load()
    assert prefix(lib, **bad) == want and "spd_shared_prefix_attn" in N.last_error()


@pytest.mark.parametrize("want,bad", [
    (UNSUPPORTED, dict(dtype=F32)), (INVALID, dict(n=-1)), (INVALID, dict(B=-1)), (INVALID, dict(S=-1)), (INVALID, dict(T=-1)),
    (INVALID, dict(Hq=3, Hkv=2)), (INVALID, dict(cu=None)), (INVALID, dict(B=3)), (UNSUPPORTED, dict(D=136)), (UNSUPPORTED, dict(D=12)),
    (UNSUPPORTED, dict(Hq=256)), (INVALID, dict(scale=0.0)), (INVALID, dict(q=None)), (INVALID, dict(k=None)), (INVALID, dict(v=None)),
    (INVALID, dict(lens=None)), (INVALID, dict(out=None)), (INVALID, dict(S=0, B=0, n=4, slots=P) | dict(B=1)), (INVALID, dict(T=0)),
    (INVALID, dict(st=60)), (INVALID, dict(sh=-8)), (INVALID, dict(sb=4)), (INVALID, dict(k=P + 2)), (INVALID, dict(ws=P + 8)),
    (UNSUPPORTED, dict(n=1 << 24, B=2, Hq=4096, Hkv=4096, T=1 << 20)),
])
def test_cross_refusals(want, bad):
    lib = N.load()
    assert cross(lib, **bad) == want and "spd_cross_attn_packed" in N.last_error()


@pytest.mark.parametrize("want,bad", [
    (UNSUPPORTED, dict(dtype=99)), (INVALID, dict(rows=-1)), (INVALID, dict(cols=0, ld=0)), (INVALID, dict(ld=9)), (INVALID, dict(x=None)),
    (INVALID, dict(u=None)), (INVALID, dict(out=None)), (INVALID, dict(x=P + 1)), (INVALID, dict(x=P + 2, dtype=F32)),
    (UNSUPPORTED, dict(cols=(1 << 19) + 1, ld=1 << 20)), (UNSUPPORTED, dict(cols=1 << 19, ld=1 << 19, dtype=F32)),
])
def test_sample_refusals(want, bad):
    lib = N.load()
    assert sample(lib, **bad) == want and "spd_sample_rows" in N.last_error()


def test_calls_without_work_return():
    lib = N.load()
    assert prefix(lib, B=0, q=None, out=None) == N.SPD_OK
    assert cross(lib, n=0, q=None, out=None) == N.SPD_OK and cross(lib, B=0, q=None, lens=None) == N.SPD_OK
    assert sample(lib, rows=0, x=None, u=None, out=None) == N.SPD_OK


def test_cpu_tensors_and_misuse_are_refused():
    q, pool = torch.zeros(3, 2, 64).half(), torch.zeros(4, 16, 2, 64).half()
    tab, ints, cu = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32)
    kv, x, u = torch.zeros(3, 2, 10, 64).half(), torch.zeros(3, 10), torch.zeros(3)
    calls = (lambda: ops.shared_prefix_decode_attention(q, pool, pool, tab[:1], ints[:1], cu, tab, ints),
             lambda: ops.shared_prefix_decode_attention(q, pool, pool, None, None, None, tab, ints),
             lambda: ops.cross_attention_packed(q, kv, kv, ints), lambda: ops.sample_rows(x, u),
             lambda: ops.sample_rows(x, u, temperature=u))
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA tensors required"):
            call()
    for call in (lambda: ops.sample_rows(None, u), lambda: ops.cross_attention_packed(q, None, kv, ints),
                 lambda: ops.shared_prefix_decode_attention(q, pool, 3, None, None, None, tab, ints)):
        with pytest.raises(RuntimeError, match="must be a tensor"):
            call()
    for name in ("shared_prefix_decode_attention", "cross_attention_packed", "sample_rows"):
        with pytest.raises(RuntimeError, match="arguments expected"):
            getattr(N.binding(), name)(q)
