"""The torch binding of the rotary, 4-bit-cache and prompt operators loads without a GPU, takes
no CPU tensors, and turns every misuse into a RuntimeError."""
import pytest
import torch

from speech_serving import _native as N
from speech_serving import ops


def _args():
    k = torch.zeros(3, 2, 64, dtype=torch.float16)
    cos = torch.ones(8, 32)
    tab = torch.zeros(3, 1, dtype=torch.int32)
    pos = torch.zeros(3, dtype=torch.int32)
    return k, cos, tab, pos


def test_cpu_tensors_are_refused():
    k, cos, tab, pos = _args()
    kp = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    pool = ops.kv_pool_int4(4, 2, 64, 16, device="cpu")
    cu = torch.tensor([0, 3], dtype=torch.int32)
    for call in (lambda: ops.rope_kv_append(k, k, k, cos, cos, kp, kp, tab, pos),
                 lambda: ops.rope_kv_append_int4(k, k, k, cos, cos, pool, tab, pos),
                 lambda: ops.kv_gather_int4(pool, tab[:1], cu, 3, 64, torch.float16),
                 lambda: ops.paged_decode_attention_int4(k, pool, tab, pos),
                 lambda: ops.prompt_attention(k, k, k, cu)):
        with pytest.raises(RuntimeError, match="CUDA tensors required"):
            call()


def test_misuse_is_a_runtime_error():
    k, cos, tab, pos = _args()
    b = N.binding()
    with pytest.raises(RuntimeError, match="must be a tensor"):
        ops.rope_kv_append(None, [1.0], k, cos, cos, k, k, tab, pos)
    with pytest.raises(RuntimeError, match="arguments expected"):
        b.prompt_attention(k, k, k)
    with pytest.raises(RuntimeError, match="no address"):
        b.setup({})
    b.setup({name: N.C.cast(getattr(N.load(), name), N.C.c_void_p).value for name in N.exported_symbols()})


def test_page_bytes_and_pools():
    lib = N.load()
    for D in (64, 128, 256):
        for bs in (8, 16, 32):
            want = 2 * (D // 64) * bs * (32 + 4)  # 4.5 bits a value, keys and values
            assert lib.spd_kv_int4_page_bytes(D, bs) == want and want % 16 == 0
            assert ops.kv_pool_int4(5, 3, D, bs, device="cpu").shape == (5, 3, want)
    for D, bs in ((96, 16), (64, 24), (0, 16), (-64, 8)):
        assert lib.spd_kv_int4_page_bytes(D, bs) == 0
        with pytest.raises(RuntimeError, match="not supported"):
            ops.kv_pool_int4(1, 1, D, bs, device="cpu")


def test_abi_refuses_bad_arguments_without_a_device():
    """Host-side checks of the C entry points come before any CUDA call."""
    lib = N.load()
    z = None
    assert lib.spd_prompt_attn(z, 0, 0, z, 0, 0, z, 0, 0, z, z, z, 1, 1, 1, 2, 1, 64, 1, 1.0, N.SPD_F32, z, z) == N.SPD_ERR_UNSUPPORTED
    assert lib.spd_prompt_attn(z, 0, 0, z, 0, 0, z, 0, 0, z, z, z, 1, 1, 1, 3, 2, 64, 1, 1.0, N.SPD_F16, z, z) == N.SPD_ERR_INVALID_ARG
    assert lib.spd_prompt_attn(z, 0, 0, z, 0, 0, z, 0, 0, z, z, z, 1, 1, 1, 2, 1, 64, 1, 1.0, N.SPD_F16, z, z) == N.SPD_ERR_INVALID_ARG
    assert "null" in N.last_error()
    assert lib.spd_kv_gather_int4(z, z, z, z, z, z, 1, 1, 1, 96, 16, 1, 1, N.SPD_F16, z, z) == N.SPD_ERR_UNSUPPORTED
    assert lib.spd_paged_decode_attn_int4(z, z, z, z, z, 1, 3, 2, 64, 16, 1, 1, 1.0, N.SPD_F16, z, 0, z) == N.SPD_ERR_INVALID_ARG
    assert lib.spd_rope_kv_append_int4(z, 0, 0, z, 0, 0, z, 0, 0, z, z, z, z, z, z, z, *([1] * 11), 7, z, z) == N.SPD_ERR_UNSUPPORTED
